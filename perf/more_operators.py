"""Attention blocks trained in 16 bits, as timed cases.

The kinds, each through the entry points that a program calls:

- ``dropout``: rows times a mask that a counter-based generator makes anew in
  each call, onto a residual or not (``layer.dropout_rows``; without a residual
  it is its own backward);
- ``attn_fwd``: softmax attention over each atom's tokens in bf16 or fp16, with
  shared key and value heads, a learned bias by buckets of the tokens' relative
  positions and dropout of the probabilities (``attention.attn_fwd_typed``);
- ``attn_bwd``: its backward, which recomputes the probabilities and the mask:
  the adjoints of q, k and v, of the cutoff factors and of the bias table
  (``attention.attn_bwd_typed``).

Atom n's tokens are row n and rows N + off[n] .. N + off[n + 1] - 1; key k
weighs exp(scale q.k + bias) cf[k], a key with cf 0 is left out and a query on
an edge with cf 0 gives zeros. ``ml`` holds each query's largest logit and the
reciprocal of its sum, zeros where no token or no key is. ``pad`` is the rows'
leading dimension past their width, ``dead`` rows of capacity past the last edge
(zeroed in the outputs), ``live`` (where not 0) the rows that count, a number the
device holds, of a buffer with capacity for more. Two int64 on the device, a seed and a step, and
the call's own number give the mask: Threefry-2x32 of 13 rounds (Salmon et al.,
2011), keyed with what it makes of (step, call) under the seed, gives four 16-bit
numbers a block; an element is left out where its number is under 65536 p.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CALL = 3


def listed():
    return [
        # one molecule's node features in fp16 onto their residual: the smallest call, where the launch counts
        {"name": "dropout-fp16-small", "kind": "dropout", "rows": 75, "width": 128, "dtype": "fp16", "p": 0.1,
         "residual": True, "pad": 0, "live": 0},
        # the tokens of the 32-structure batch at d 512 after the output projection, onto the residual
        {"name": "dropout-batch-bf16", "kind": "dropout", "rows": 498338, "width": 512, "dtype": "bf16", "p": 0.1,
         "residual": True, "pad": 0, "live": 0},
        # the backward of an odd width in a wider buffer, with capacity rows past the live ones
        {"name": "dropout-odd-fp32", "kind": "dropout", "rows": 62291, "width": 333, "dtype": "fp32", "p": 0.25,
         "residual": False, "pad": 1, "live": 62001},
        # one molecule: nine atoms, 4 heads of 32; the smallest call
        {"name": "attn-fwd-small-fp16", "kind": "attn_fwd", "atoms": 9, "least_edges": 4, "most_edges": 8, "heads": 4,
         "kv_heads": 4, "head_dim": 32, "dtype": "fp16", "buckets": 32, "reach": 128, "p": 0.0, "zeros": 0.0,
         "pad": 0, "dead": 0},
        # the 1728-atom diamond (70 edges an atom) at d 256: the plain attention
        {"name": "attn-fwd-diamond-bf16", "kind": "attn_fwd", "atoms": 1728, "least_edges": 70, "most_edges": 70,
         "heads": 8, "kv_heads": 8, "head_dim": 32, "dtype": "bf16", "buckets": 0, "reach": 0, "p": 0.0, "zeros": 0.0,
         "pad": 0, "dead": 0},
        # the 32-structure batch at d 512 in training: bias over the edges' shells, dropout of the probabilities
        {"name": "attn-fwd-batch-bf16", "kind": "attn_fwd", "atoms": 11392, "least_edges": 31, "most_edges": 70,
         "heads": 8, "kv_heads": 8, "head_dim": 64, "dtype": "bf16", "buckets": 32, "reach": 128, "p": 0.1,
         "zeros": 0.05, "pad": 0, "dead": 0},
        # two whole structures attended to at once, tokens in order, four heads to a key head
        {"name": "attn-fwd-long-bf16", "kind": "attn_fwd", "atoms": 2, "least_edges": 3500, "most_edges": 4095,
         "heads": 8, "kv_heads": 2, "head_dim": 128, "dtype": "bf16", "buckets": 32, "reach": 128, "p": 0.0,
         "zeros": 0.0, "pad": 0, "dead": 0},
        # and their backwards
        {"name": "attn-bwd-small-fp16", "kind": "attn_bwd", "atoms": 9, "least_edges": 4, "most_edges": 8, "heads": 4,
         "kv_heads": 4, "head_dim": 32, "dtype": "fp16", "buckets": 32, "reach": 128, "p": 0.0, "zeros": 0.0,
         "pad": 0, "dead": 0},
        {"name": "attn-bwd-diamond-bf16", "kind": "attn_bwd", "atoms": 1728, "least_edges": 70, "most_edges": 70,
         "heads": 8, "kv_heads": 8, "head_dim": 32, "dtype": "bf16", "buckets": 0, "reach": 0, "p": 0.0, "zeros": 0.0,
         "pad": 0, "dead": 0},
        {"name": "attn-bwd-batch-bf16", "kind": "attn_bwd", "atoms": 11392, "least_edges": 31, "most_edges": 70,
         "heads": 8, "kv_heads": 8, "head_dim": 64, "dtype": "bf16", "buckets": 32, "reach": 128, "p": 0.1,
         "zeros": 0.05, "pad": 0, "dead": 0},
        {"name": "attn-bwd-long-bf16", "kind": "attn_bwd", "atoms": 2, "least_edges": 3500, "most_edges": 4095,
         "heads": 8, "kv_heads": 2, "head_dim": 128, "dtype": "bf16", "buckets": 32, "reach": 128, "p": 0.0,
         "zeros": 0.0, "pad": 0, "dead": 0},
        # counts from a lone atom to 300 tokens, a head_dim that fills no tile, wider rows, capacity, edges at the
        # cutoff
        {"name": "attn-bwd-odd-fp16", "kind": "attn_bwd", "atoms": 301, "least_edges": 0, "most_edges": 299,
         "heads": 6, "kv_heads": 3, "head_dim": 24, "dtype": "fp16", "buckets": 17, "reach": 50, "p": 0.25,
         "zeros": 0.1, "pad": 3, "dead": 37},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["dropout", "attn_fwd", "attn_fwd", "attn_bwd", "attn_bwd", "attn_bwd"])
    p = rng.choice([0.0, 0.05, 0.1, 0.25, 0.5])
    if kind == "dropout":
        width = _log_int(rng, 16, 16384)
        if rng.random() < 0.5:
            width = max(16, width // 16 * 16)
        rows = _log_int(rng, 1, min(498338, (1 << 26) // width))
        return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "p": p or 0.1, "residual": rng.random() < 0.6, "pad": rng.choice([0, 0, 0, 1, 8]),
                "live": rng.randint(1, rows) if rng.random() < 0.25 else 0}
    heads, group = rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 1, 1, 2, 4])
    heads = heads if heads % group == 0 else heads * group
    head_dim = rng.choice([16, 24, 32, 32, 32, 40, 64, 64, 64, 80, 96, 128])
    most = _log_int(rng, 4, 4096)  # the longest atom's tokens
    cells = min(57_000_000, 440_000_000 // heads, 28_000_000_000 // (heads * head_dim))
    atoms = _log_int(rng, 1, max(1, min(12000, cells // most ** 2, 250_000_000 // (most * heads * head_dim))))
    spread = rng.choice([0.0, 0.5, 1.0])
    buckets = rng.choice([0, 17, 32, 32, 64])
    return {"kind": kind, "atoms": atoms, "least_edges": round((most - 1) * (1 - spread)), "most_edges": most - 1,
            "heads": heads,
            "kv_heads": heads // group, "head_dim": head_dim, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "buckets": buckets, "reach": rng.choice([50, 128, 512]) if buckets else 0, "p": rng.choice([0.0, p]),
            "zeros": rng.choice([0.0, 0.0, 0.1]), "pad": rng.choice([0, 0, 0, 1, 8]),
            "dead": rng.choice([0, 0, 37])}


# ---- inputs -------------------------------------------------------------------------


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(device=_device()).manual_seed(seed)


def _rows(gen, rows, width, pad, dtype, spread, size=1.0):
    """[rows, width] of normals in a buffer `pad` columns wider; every column's
    size is its own (log-normal), as features and their adjoints have them."""
    dev = _device()
    x = torch.empty((rows, width + pad), dtype=dtype, device=dev)[:, :width]
    col = size * torch.exp(spread * torch.randn(width, generator=gen, device=dev))
    step = max(1, (1 << 26) // width)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        x[r:r + n] = (torch.randn((n, width), generator=gen, device=dev) * col).to(dtype)
    return x


def _layout(case):
    """The atoms' edge counts (the first atom has the most), and which edges lie at the cutoff."""
    rng = np.random.default_rng(case["atoms"])
    lo, hi = case["least_edges"], case["most_edges"]
    counts = rng.integers(lo, hi + 1, size=case["atoms"])
    counts[0] = hi
    return counts, rng.random(int(counts.sum())) < case["zeros"]


def _sizes(case):
    """(T with its dead rows, S, q's columns, all of q, k and v's)."""
    counts, _ = _layout(case)
    wide = case["heads"] * case["head_dim"]
    return (case["atoms"] + int(counts.sum()) + case["dead"], case["most_edges"] + 1, wide,
            wide + 2 * case["kv_heads"] * case["head_dim"])


def _bucket_table(n, reach):
    """The bucket of each offset -reach .. reach (key's position less the
    query's): half of the buckets to each sign, of a half the first half one to an
    offset, the rest at equal ratios up to reach (in whole numbers, which have no
    rounding at a border)."""
    half = n // 2
    single = max(1, half // 2)
    wide = half - single
    table = []
    for offset in range(-reach, reach + 1):
        d, b = abs(offset), abs(offset)
        if d >= single:
            b = single
            while b < half - 1 and d ** wide * single ** (b + 1 - single) >= reach ** (b + 1 - single) * single ** wide:
                b += 1
        table.append(b + (half if offset > 0 else 0))
    return table


def prepare(case, seed):
    gen, dev = _generator(seed), _device()
    dtype = DTYPES[case["dtype"]]
    state = {"case": case, "rng": torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 63), 1000 + seed % 977],
                                               dtype=torch.int64, device=dev)}
    if case["kind"] == "dropout":
        rows, width = case["rows"], case["width"]
        state["inp"] = _rows(gen, rows, width, case["pad"], dtype, 0.5)
        state["residual"] = _rows(gen, rows, width, case["pad"], dtype, 0.5) if case["residual"] else None
        state["out"] = torch.zeros((rows, width), dtype=dtype, device=dev)
        state["live"] = torch.tensor([case["live"]], dtype=torch.int32, device=dev) if case["live"] else None
        return state
    counts, zero = _layout(case)
    N, E, (T, S, D, W) = case["atoms"], int(counts.sum()), _sizes(case)
    off = np.zeros(N + 1, dtype=np.int32)
    off[1:] = np.cumsum(counts)
    state["off"] = torch.from_numpy(off).to(dev)
    state["qkv"] = _rows(gen, T, W, case["pad"], dtype, 0.3)
    cut = 0.05 + 0.95 * torch.rand(E, generator=gen, device=dev)
    cut[torch.from_numpy(zero).to(dev)] = 0.0
    slot = torch.arange(S, device=dev)[None, :]
    at = state["off"][:N, None].long() + slot - 1
    edge = (slot > 0) & (slot <= torch.from_numpy(counts).to(dev)[:, None])
    state["cf"] = torch.where(edge, cut[at.clamp(0, max(E - 1, 0))] if E else 0.0, (slot == 0).float()).contiguous()
    if case["buckets"]:
        state["table"] = 0.5 * torch.randn((case["buckets"], case["heads"]), generator=gen, device=dev)
        state["buckets"] = torch.tensor(_bucket_table(case["buckets"], case["reach"]), dtype=torch.int32, device=dev)
        # long neighbourhoods are in order, short ones have their edges' radial shells
        pos = torch.randint(0, 160, (T,), generator=gen, device=dev, dtype=torch.int32)
        if S > 512:
            pos[N:] = torch.arange(T - N, device=dev, dtype=torch.int32)
            pos[:N] = state["off"][:N]
        else:
            pos[:N] = 0
        state["pos"] = pos
    state["merged"] = torch.zeros((T, D), dtype=dtype, device=dev)
    state["ml"] = torch.zeros((N * case["heads"] * S, 2), device=dev)
    if case["kind"] == "attn_bwd":
        out, top, inv = _forward(state)[:3]
        state["merged"] = out
        state["ml"] = torch.stack([top, inv], -1).view(-1, 2).contiguous()
        state["dmerged"] = _rows(gen, T, D, case["pad"], dtype, 0.3, 1e-2)
        state["qkv_adj"] = torch.zeros((T, W), dtype=dtype, device=dev)
        state["cf_adj"] = torch.zeros((N, S), device=dev)
        state["table_adj"] = torch.zeros_like(state["table"]) if case["buckets"] else None
    return state


# ---- the pass -----------------------------------------------------------------------

LOW = 0xFFFFFFFF
TURNS = (13, 15, 26, 6, 17, 29, 16, 24)


def _threefry(k0, k1, x, y):
    """Threefry-2x32, 13 rounds, of int64 tensors that hold 32-bit words."""
    keys = (k0, k1, k0 ^ k1 ^ 0x1BD11BDA)
    x, y = (x + keys[0]) & LOW, (y + keys[1]) & LOW
    for i in range(13):
        x = (x + y) & LOW
        turn = TURNS[i % 8]
        y = (((y << turn) | (y >> (32 - turn))) & LOW) ^ x
        if i % 4 == 3:
            j = (i + 1) // 4
            x, y = (x + keys[j % 3]) & LOW, (y + keys[(j + 1) % 3] + j) & LOW
    return x, y


def _kept(state, x, y, n):
    """Which elements stay: the last axis' n, four to each of the counters (x, y)."""
    rng, p = state["rng"], state["case"]["p"]
    k0, k1 = _threefry(rng[0] & LOW, (rng[0] >> 32) & LOW, rng[1] & LOW, torch.full_like(rng[1], CALL))
    a, b = _threefry(k0, k1, x, y)
    words = torch.stack([a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16], -1).flatten(-2)
    return words[..., :n] >= round(65536 * p)


def _tokens(state):
    """(rows [N, S], which slots are tokens, which keys count, which queries do)."""
    N, S = state["cf"].shape
    slot = torch.arange(S, device=state["cf"].device)[None, :]
    off = state["off"].long()
    rows = torch.where(slot == 0, torch.arange(N, device=slot.device)[:, None], N + off[:-1, None] + slot - 1)
    there = slot <= (off[1:] - off[:-1])[:, None]
    keys = there & (state["cf"] > 0)
    return torch.where(there, rows, 0), there, keys, keys | (slot == 0)


def _heads(x, rows, mask, count, head_dim):
    """[N, count, S, head_dim] in fp32 of the rows' columns, zeros where not masked in."""
    got = torch.where(mask[:, :, None], x[rows].float(), 0.0)
    return got.view(*rows.shape, count, head_dim).transpose(1, 2).contiguous()


def _forward(state):
    case = state["case"]
    H, G, hd, kv = case["heads"], case["heads"] // case["kv_heads"], case["head_dim"], case["kv_heads"]
    rows, there, keys, queries = _tokens(state)
    N, S = rows.shape
    D = H * hd
    qkv = state["qkv"]
    q = _heads(qkv[:, :D], rows, queries, H, hd)
    k = _heads(qkv[:, D:D + kv * hd], rows, keys, kv, hd).repeat_interleave(G, 1)
    v = _heads(qkv[:, D + kv * hd:], rows, keys, kv, hd).repeat_interleave(G, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    bucket = None
    if case["buckets"]:
        pos = state["pos"][rows]
        bucket = state["buckets"][(pos[:, None, :] - pos[:, :, None]).clamp(-case["reach"], case["reach"])
                                  + case["reach"]].long()
        s = s + state["table"][bucket].permute(0, 3, 1, 2)
    s = s + torch.log(state["cf"])[:, None, None, :]
    s = torch.where(keys[:, None, None, :], s, -math.inf)
    full = (queries & keys.any(1, keepdim=True))[:, None, :]
    top = torch.where(full, s.amax(-1), 0.0)
    e = torch.exp(s - top[..., None])
    total = e.sum(-1)
    inv = torch.where(full, 1.0 / total, 0.0)
    prob = e * inv[..., None]
    keep = None
    if case["p"]:
        group = torch.arange((S + 3) // 4, device=s.device)
        keep = _kept(state, rows[:, None, :, None], group * H + torch.arange(H, device=s.device)[None, :, None, None],
                     S) * (65536.0 / (65536 - round(65536 * case["p"])))
    out = torch.matmul(prob if keep is None else prob * keep, v)
    merged = torch.zeros((qkv.shape[0], D), dtype=qkv.dtype, device=qkv.device)
    merged[rows[there]] = out.transpose(1, 2).reshape(N, S, D)[there].to(qkv.dtype)
    return merged, top, inv, prob, keep, (q, k, v), bucket


def _backward(state):
    case = state["case"]
    H, G, hd, kv = case["heads"], case["heads"] // case["kv_heads"], case["head_dim"], case["kv_heads"]
    _, _, _, prob, keep, (q, k, v), bucket = _forward(state)
    rows, there, keys, queries = _tokens(state)
    N, S = rows.shape
    D, scale = H * hd, 1.0 / math.sqrt(hd)
    do = _heads(state["dmerged"], rows, queries, H, hd)
    o = _heads(state["merged"], rows, queries, H, hd)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    if keep is not None:
        dp = dp * keep
    ds = prob * (dp - (do * o).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * scale
    dv = torch.matmul((prob if keep is None else prob * keep).transpose(2, 3).contiguous(), do)
    dk, dv = (x.view(N, kv, G, S, hd).sum(2) for x in (dk, dv))
    qkv_adj = torch.zeros((state["qkv"].shape[0], D + 2 * kv * hd), dtype=state["qkv"].dtype, device=ds.device)
    flat = torch.cat([x.transpose(1, 2).reshape(N, S, -1) for x in (dq, dk, dv)], -1)
    qkv_adj[rows[there]] = flat[there].to(qkv_adj.dtype)
    cf = state["cf"]
    got = {"qkv_adj": qkv_adj, "cf_adj": torch.where(keys, ds.sum((1, 2)) / torch.where(keys, cf, 1.0), 0.0)}
    if bucket is not None:
        marks = (bucket[..., None] == torch.arange(case["buckets"], device=ds.device)).float()
        each = torch.matmul(ds.transpose(1, 2).reshape(N * S, H, S), marks.view(N * S, S, -1))
        got["table_adj"] = each.double().sum(0).t().contiguous().float()
    return got


def _plain(state):
    case = state["case"]
    if case["kind"] == "attn_fwd":
        merged, top, inv = _forward(state)[:3]
        return {"merged": merged, "ml": torch.stack([top, inv], -1).view(-1, 2)}
    if case["kind"] == "attn_bwd":
        return _backward(state)
    inp = state["inp"]
    row = torch.arange(case["rows"], device=inp.device)[:, None]
    group = torch.arange((case["width"] + 3) // 4, device=inp.device)[None, :]
    keep = _kept(state, row, group, case["width"])
    y = torch.where(keep, inp.float() * (65536.0 / (65536 - round(65536 * case["p"]))), 0.0)
    if state["residual"] is not None:
        y = state["residual"].float() + y
    y = y.to(inp.dtype)
    return y if state["live"] is None else torch.where(row < state["live"], y, state["out"])


def run(state):
    if not own:
        return _plain(state)
    from pet_kokkos_amd import attention, layer
    case = state["case"]
    drop = attention.Dropout(case["p"], state["rng"], CALL) if case["p"] else None
    if case["kind"] == "dropout":
        layer.dropout_rows(state["out"], state["inp"], drop, residual=state["residual"], live=state["live"])
        return state["out"]
    bias = attention.RelativeBias(state["table"], state["buckets"], state["pos"]) if case["buckets"] else None
    if case["kind"] == "attn_fwd":
        attention.attn_fwd_typed(state["qkv"], state["off"], state["cf"], case["heads"], case["head_dim"],
                                 kv_heads=case["kv_heads"], bias=bias, dropout=drop, dead=case["dead"] > 0,
                                 merged=state["merged"], ml=state["ml"])
        return {"merged": state["merged"], "ml": state["ml"]}
    attention.attn_bwd_typed(state["qkv"], state["off"], state["dmerged"], state["merged"], state["ml"], state["cf"],
                             case["heads"], case["head_dim"], kv_heads=case["kv_heads"], bias=bias, dropout=drop,
                             dead=case["dead"] > 0, qkv_adj=state["qkv_adj"], cf_seq_adj=state["cf_adj"],
                             bias_adj=state["table_adj"])
    got = {"qkv_adj": state["qkv_adj"], "cf_adj": state["cf_adj"]}
    if bias is not None:
        got["table_adj"] = state["table_adj"]
    return got


# ---- the work and the definition ----------------------------------------------------


def work(case):
    if case["kind"] == "dropout":
        live, size = case["live"] or case["rows"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": (3 if case["residual"] else 2) * live * case["width"] * size + 16,
                "flops": (2 if case["residual"] else 1) * live * case["width"]}
    counts, zero = _layout(case)
    T, S, D, W = _sizes(case)
    T -= case["dead"]
    first = np.zeros(len(counts) + 1, dtype=np.int64)
    first[1:] = np.cumsum(counts)
    at_cutoff = np.concatenate([[0], np.cumsum(zero)])
    live = 1 + counts - (at_cutoff[first[1:]] - at_cutoff[first[:-1]])
    pairs = int((live.astype(np.int64) ** 2).sum()) * case["heads"]
    small = 4 * (case["atoms"] + 1) + 4 * T + 8 * case["heads"] * T
    if case["buckets"]:
        small += 4 * T + 4 * case["buckets"] * case["heads"] * (1 if case["kind"] == "attn_fwd" else 2)
    if case["kind"] == "attn_fwd":
        return {"bytes": 2 * T * (W + D) + small, "flops": 4 * pairs * case["head_dim"]}
    return {"bytes": 2 * T * (2 * W + 2 * D) + small + 4 * T, "flops": 10 * pairs * case["head_dim"]}


def _words(seed, step, x, y):
    """The generator once more, of int32 tensors that wrap: the two words of (x, y)."""

    def turn(v, r):
        return (v << r) | ((v >> (32 - r)) & ((1 << r) - 1))

    def signed(v):
        return v - (1 << 32) if v >= 1 << 31 else v

    def block(k0, k1, x, y):
        if isinstance(k0, int):
            k0, k1 = torch.tensor([signed(k0)], dtype=torch.int32, device=x.device), torch.tensor(
                [signed(k1)], dtype=torch.int32, device=x.device)
        k2 = k0 ^ k1 ^ 0x1BD11BDA
        x, y = x + k0, y + k1
        for r in (13, 15, 26, 6):
            x = x + y
            y = turn(y, r) ^ x
        x, y = x + k1, y + k2 + 1
        for r in (17, 29, 16, 24):
            x = x + y
            y = turn(y, r) ^ x
        x, y = x + k2, y + k0 + 2
        for r in (13, 15, 26, 6):
            x = x + y
            y = turn(y, r) ^ x
        x, y = x + k0, y + k1 + 3
        x = x + y
        return x, turn(y, 17) ^ x

    one = torch.tensor([signed(step & LOW)], dtype=torch.int32, device=x.device)
    k0, k1 = block(seed & LOW, (seed >> 32) & LOW, one, torch.full_like(one, CALL))
    return block(k0, k1, x, y)


def _mask64(state, x, y, n):
    """1 / (1 - p) where an element stays, else 0, in 64 bits; x and y int32, the last axis the counters'."""
    least = round(65536 * state["case"]["p"])
    a, b = _words(int(state["rng"][0]), int(state["rng"][1]), x, y)
    got = torch.empty((*a.shape, 4), dtype=torch.float64, device=a.device)
    for i, w in enumerate((a, a >> 16, b, b >> 16)):
        got[..., i] = ((w & 0xFFFF) >= least).double()
    return got.reshape(*a.shape[:-1], -1)[..., :n] / (1.0 - least / 65536.0)


def exact(case, seed):
    state = prepare(case, seed)
    dev = _device()
    if case["kind"] == "dropout":
        res = torch.zeros((case["rows"], case["width"]), dtype=torch.float64, device=dev)
        live = case["live"] or case["rows"]
        step = max(1, (1 << 25) // case["width"])
        group = torch.arange((case["width"] + 3) // 4, device=dev, dtype=torch.int32)[None, :]
        for r in range(0, live, step):
            at = slice(r, min(live, r + step))
            row = torch.arange(at.start, at.stop, device=dev, dtype=torch.int32)[:, None]
            res[at] = state["inp"][at].double() * _mask64(state, row.expand(-1, group.shape[1]),
                                                          group.expand(row.shape[0], -1), case["width"])
            if state["residual"] is not None:
                res[at] += state["residual"][at].double()
        return res
    H, hd, kv = case["heads"], case["head_dim"], case["kv_heads"]
    N, (T, S, D, W) = case["atoms"], _sizes(case)
    counts, _ = _layout(case)
    first = np.concatenate([[0], np.cumsum(counts)])
    back = case["kind"] == "attn_bwd"
    merged = torch.zeros((T, D), dtype=torch.float64, device=dev)
    ml = torch.zeros((N, H, S, 2), dtype=torch.float64, device=dev)
    adj = torch.zeros((T, W), dtype=torch.float64, device=dev) if back else None
    cf_adj = torch.zeros((N, S), dtype=torch.float64, device=dev)
    table_adj = torch.zeros((case["buckets"], H), dtype=torch.float64, device=dev)
    # atoms of like counts together, each padded to the group's longest; a head at a time
    order = np.argsort(counts, kind="stable")
    most = max(1, (1 << 26) // S ** 2)
    for g in range(0, N, most):
        atoms = order[g:g + most]
        n, L = len(atoms), int(counts[atoms].max()) + 1
        rows = np.zeros((n, L), dtype=np.int64)
        slot = np.arange(L)[None, :]
        rows[:] = np.where(slot == 0, atoms[:, None], N + first[atoms][:, None] + slot - 1)
        here = torch.from_numpy(slot <= counts[atoms][:, None]).to(dev)
        rows = torch.where(here, torch.from_numpy(rows).to(dev), 0)
        which = torch.from_numpy(atoms).to(dev)
        cf = state["cf"][which, :L].double() * here
        key, query = cf > 0, here & ((cf > 0) | (torch.arange(L, device=dev)[None, :] == 0))
        if case["buckets"]:
            pos = state["pos"][rows].long()
            bucket = state["buckets"][torch.clamp(pos[:, None, :] - pos[:, :, None], -case["reach"], case["reach"])
                                      + case["reach"]].long()
        for h in range(H):
            def part(x, c):
                return x[:, c * hd:(c + 1) * hd][rows].double()
            c = h // (H // kv)
            q = part(state["qkv"], h) * query[..., None]
            k = part(state["qkv"], H + c) * key[..., None]
            v = part(state["qkv"], H + kv + c) * key[..., None]
            s = torch.bmm(q, k.transpose(1, 2).contiguous()) / hd ** 0.5
            if case["buckets"]:
                s += state["table"][:, h].double()[bucket]
            s = torch.where(key[:, None, :], s + torch.log(cf)[:, None, :], -math.inf)
            top = s.max(-1, keepdim=True).values
            e = torch.exp(s - top) * query[:, :, None]
            total = e.sum(-1, keepdim=True)
            prob = torch.where(total > 0, e / total, 0.0)
            mask = 1.0
            if case["p"]:
                y = torch.arange((L + 3) // 4, device=dev, dtype=torch.int32) * H + h
                x = rows.int()[:, :, None].expand(-1, -1, len(y))
                mask = _mask64(state, x, y.expand_as(x), L)
            if not back:
                merged[rows[here], h * hd:(h + 1) * hd] = torch.bmm(prob * mask, v)[here]
                ml[which, h, :L, 0] = torch.where(query, top[..., 0], 0.0)
                ml[which, h, :L, 1] = torch.where(query, 1.0 / total[..., 0], 0.0)
                continue
            do, o = (part(state[x], h) * query[..., None] for x in ("dmerged", "merged"))
            ds = prob * (torch.bmm(do, v.transpose(1, 2).contiguous()) * mask - (do * o).sum(-1, keepdim=True))
            across = torch.arange(hd, device=dev)[None, :]
            tokens = rows[here][:, None]
            adj[tokens, h * hd + across] = (torch.bmm(ds, k) / hd ** 0.5)[here]
            adj[tokens, (H + c) * hd + across] += (torch.bmm(ds.transpose(1, 2).contiguous(), q) / hd ** 0.5)[here]
            adj[tokens, (H + kv + c) * hd + across] += torch.bmm((prob * mask).transpose(1, 2).contiguous(), do)[here]
            cf_adj[which[:, None], torch.arange(L, device=dev)[None, :]] += torch.where(key, ds.sum(1) / cf, 0.0)
            if case["buckets"]:
                for b in range(case["buckets"]):
                    table_adj[b, h] += torch.where(bucket == b, ds, 0.0).sum()
    if not back:
        return {"merged": merged, "ml": ml.view(-1, 2)}
    got = {"qkv_adj": adj, "cf_adj": cf_adj}
    if case["buckets"]:
        got["table_adj"] = table_adj
    return got
