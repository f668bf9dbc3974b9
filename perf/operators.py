"""A training step's operators, as timed cases.

The kinds, each through the entry points that a program calls:

- ``norm``: RMSNorm / LayerNorm of rows in 16 bits, or wider than 2048 columns
  (``layer.norm_rows``);
- ``norm_grads``: its backward, the rows' adjoint with the weight's and bias's
  gradients (``layer.norm_rows_grads``);
- ``linear_grads``: a dense layer's weight and bias gradients from its input
  rows and its output's adjoint (``linear.linear_grads``);
- ``grad_norm``: the norm of all of a model's gradients (``grads.grad_norm``);
- ``clip``: the same with the gradients scaled and clipped in place
  (``grads.clip_grads``).

Rows are fp32, bf16 or fp16, parameters and their gradients fp32 (gradient
lists hold any of the three). ``pad`` is the rows' leading dimension past their
width; ``live`` (where not 0) the rows that count, a number the device holds,
of a buffer with capacity for more.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
RMS_EPS = 2.0 ** -23
LN_EPS = 1e-5
MAX_NORM = 1.0


def listed():
    return [
        # one molecule's node features in fp16: the smallest call, where launches count
        {"name": "norm-fp16-small", "kind": "norm", "rows": 75, "width": 128, "dtype": "fp16", "ln": True, "pad": 0},
        # rows wider than PET's, as a model that shares its trunk with a language model has them
        {"name": "norm-bf16-wide", "kind": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "ln": False, "pad": 0},
        # the tokens of 648-atom water, d 128 (26670 edges): the norm before an attention block
        {"name": "norm-grads-water", "kind": "norm_grads", "rows": 27318, "width": 128, "dtype": "fp32", "ln": False,
         "pad": 0, "live": 0},
        # the 32-structure batch at d 512 (498338 tokens), activations kept in bf16, the residual family's LayerNorm
        {"name": "norm-grads-batch-bf16", "kind": "norm_grads", "rows": 498338, "width": 512, "dtype": "bf16",
         "ln": True, "pad": 0, "live": 0},
        # an odd width in a wider buffer, with capacity rows past the live ones
        {"name": "norm-grads-odd-fp16", "kind": "norm_grads", "rows": 10240, "width": 777, "dtype": "fp16", "ln": True,
         "pad": 3, "live": 10007},
        # the centre MLP's input layer on 648 atoms: few rows, where launches count
        {"name": "linear-grads-centre", "kind": "linear_grads", "rows": 648, "n": 1024, "k": 256, "dtype": "fp32",
         "pad": 0, "live": 0},
        # the QKV projection of the 1728-atom diamond at d 256
        {"name": "linear-grads-qkv", "kind": "linear_grads", "rows": 122688, "n": 768, "k": 256, "dtype": "fp32",
         "pad": 0, "live": 0},
        # the edge MLP's SwiGLU layer of the 32-structure batch at d 512, activations in bf16
        {"name": "linear-grads-batch-bf16", "kind": "linear_grads", "rows": 486946, "n": 2048, "k": 512,
         "dtype": "bf16", "pad": 0, "live": 0},
        # sizes that fill no tile, in wider buffers
        {"name": "linear-grads-odd", "kind": "linear_grads", "rows": 62291, "n": 500, "k": 333, "dtype": "fp32",
         "pad": 1, "live": 62001},
        # every gradient of the 128-wide model of the water benchmark (2 x 2 layers)
        {"name": "grad-norm-128", "kind": "grad_norm", "width": 128, "hidden": 512, "layers": 4, "dtypes": "fp32",
         "p": 2.0, "scale": 1.0},
        # the same model's gradients clipped after a backward whose last micro-batch was ragged
        {"name": "clip-128", "kind": "clip", "width": 128, "hidden": 512, "layers": 4, "dtypes": "fp32", "p": 2.0,
         "scale": 0.977},
        # a large model's gradients, matrices in bf16 and vectors in fp32, many times what the caches hold
        {"name": "clip-large-mixed", "kind": "clip", "width": 1280, "hidden": 5120, "layers": 12, "dtypes": "bf16",
         "p": 2.0, "scale": 0.977},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_grads", "norm_grads", "norm_grads", "linear_grads", "linear_grads",
                       "linear_grads", "grad_norm", "clip"])
    if kind in ("norm", "norm_grads"):
        width = _log_int(rng, 16, 16384)
        if rng.random() < 0.5:
            width = max(16, width // 16 * 16)
        case = {"kind": kind, "rows": _log_int(rng, 1, min(498338, (1 << 26) // width)), "width": width,
                "ln": rng.random() < 0.5, "pad": rng.choice([0, 0, 0, 1, 8])}
        # (the fp32 rows of the library's first norm end at 2048 columns: wider ones or 16 bits are new)
        dtypes = ["bf16", "fp16"] if kind == "norm" and width <= 2048 else ["fp32", "bf16", "fp16"]
        case["dtype"] = rng.choice(dtypes)
        if kind == "norm_grads":
            case["live"] = rng.randint(1, case["rows"]) if rng.random() < 0.25 else 0
        return case
    if kind == "linear_grads":
        n, k = _log_int(rng, 4, 4096), _log_int(rng, 4, 4096)
        if rng.random() < 0.6:
            n, k = max(16, n // 16 * 16), max(16, k // 16 * 16)
        most = min(498338, (1 << 38) // (n * k), (1 << 29) // max(n, k))
        rows = _log_int(rng, 1, most)
        return {"kind": kind, "rows": rows, "n": n, "k": k, "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                "pad": rng.choice([0, 0, 0, 1, 8]), "live": rng.randint(1, rows) if rng.random() < 0.25 else 0}
    width = rng.choice([64, 128, 192, 256, 320, 512, 640, 1280])
    return {"kind": kind, "width": width, "hidden": width * rng.choice([1, 2, 4]),
            "layers": rng.randint(1, 12 if width <= 640 else 6),
            "dtypes": rng.choice(["fp32", "bf16", "fp16", "mixed"]), "p": rng.choice([2.0, 2.0, 2.0, math.inf, 1.0]),
            "scale": rng.choice([1.0, 0.977]) if kind == "grad_norm" else round(rng.uniform(0.95, 0.99), 3)}


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


def _parameter_shapes(case):
    """A PET-shaped model's parameters: per layer the attention's two products,
    the edges' and the centres' MLPs, two norms, the read-out heads at the end."""
    d, f = case["width"], case["hidden"]
    e = 2 * d  # the centres' width
    shapes = []
    for _ in range(case["layers"]):
        shapes += [(3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (2 * f, d), (2 * f,), (d, f), (d,),
                   (d, e), (d,), (e, d), (e,), (e,), (4 * e, e), (4 * e,), (e, 2 * e), (e,)]
    return shapes + [(128, e), (128,), (128, 128), (128,), (1, 128), (1,), (128, d), (128,), (128, 128), (128,),
                     (1, 128), (1,)]


def _grad_dtype(case, i, shape):
    """Parameter i's gradient: matrices in the case's type (or each of the three in turn), vectors in fp32."""
    if len(shape) == 1:
        return "fp32"
    return ["fp32", "bf16", "fp16"][i % 3] if case["dtypes"] == "mixed" else case["dtypes"]


def prepare(case, seed):
    gen, dev, kind = _generator(seed), _device(), case["kind"]
    state = {"case": case}
    if kind in ("norm", "norm_grads"):
        rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        state["inp"] = _rows(gen, rows, width, case["pad"], dtype, 0.5)
        state["weight"] = 1.0 + 0.1 * torch.randn(width, generator=gen, device=dev)
        state["bias"] = 0.1 * torch.randn(width, generator=gen, device=dev) if case["ln"] else None
        state["out"] = torch.zeros((rows, width), dtype=dtype, device=dev)
        if kind == "norm_grads":
            state["out_adj"] = _rows(gen, rows, width, case["pad"], dtype, 0.5, 1e-2)
            state["w_adj"] = torch.zeros(width, device=dev)
            state["b_adj"] = torch.zeros(width, device=dev) if case["ln"] else None
    elif kind == "linear_grads":
        dtype = DTYPES[case["dtype"]]
        state["out_adj"] = _rows(gen, case["rows"], case["n"], case["pad"], dtype, 1.0, 1e-2)
        state["inp"] = _rows(gen, case["rows"], case["k"], case["pad"], dtype, 0.5)
        state["w_adj"] = torch.zeros((case["n"], case["k"]), device=dev)
        state["b_adj"] = torch.zeros(case["n"], device=dev)
    else:
        # the gradients are views of one flat buffer a type, as a trainer that shares them out keeps them
        shapes = _parameter_shapes(case)
        dtypes = [_grad_dtype(case, i, shape) for i, shape in enumerate(shapes)]
        state["flat"] = {}
        for name, dtype in DTYPES.items():
            count = sum(math.prod(shape) for shape, d in zip(shapes, dtypes) if d == name)
            if count:
                state["flat"][name] = torch.empty(count, dtype=dtype, device=dev)
        at, grads = dict.fromkeys(DTYPES, 0), []
        sizes = torch.randn(len(shapes), generator=torch.Generator().manual_seed(seed))
        for shape, name, size in zip(shapes, dtypes, sizes.exp().tolist()):
            g = state["flat"][name][at[name]:at[name] + math.prod(shape)].view(shape)
            g.copy_(1e-2 * size * torch.randn(shape, generator=gen, device=dev))
            at[name] += math.prod(shape)
            grads.append(g)
        state["grads"] = grads
        if own:
            from pet_kokkos_amd import grads as gr
            state["list"] = gr.GradList(grads)
    if case.get("live"):
        state["live"] = torch.tensor([case["live"]], dtype=torch.int32, device=dev)
    else:
        state["live"] = None
    return state


# ---- the pass -----------------------------------------------------------------------


def _norm_parts(x, ln):
    if ln:
        x = x - x.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + (LN_EPS if ln else RMS_EPS))
    return x * inv, inv


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "norm":
        xhat, _ = _norm_parts(state["inp"].float(), case["ln"])
        y = xhat * state["weight"]
        if case["ln"]:
            y = y + state["bias"]
        state["out"].copy_(y)
        return state["out"]
    if kind in ("norm_grads", "linear_grads"):
        x, g = state["inp"].float(), state["out_adj"].float()
        keep = None
        if state["live"] is not None:
            keep = (torch.arange(case["rows"], device=x.device) < state["live"])[:, None]
            x, g = torch.where(keep, x, 0.0), torch.where(keep, g, 0.0)
        if kind == "linear_grads":
            return {"w_adj": g.t() @ x, "b_adj": g.sum(0)}
        xhat, inv = _norm_parts(x, case["ln"])
        gw = g * state["weight"]
        d = gw - xhat * (gw * xhat).mean(1, keepdim=True)
        if case["ln"]:
            d = d - gw.mean(1, keepdim=True)
        d = (inv * d).to(state["inp"].dtype)
        got = {"in_adj": d if keep is None else torch.where(keep, d, state["out"]), "w_adj": (g * xhat).sum(0)}
        if case["ln"]:
            got["b_adj"] = g.sum(0)
        return got
    p, scale = case["p"], case["scale"]
    if p == 2.0:
        parts = [(g.double() ** 2).sum() for g in state["grads"]]
        norm = scale * torch.sqrt(torch.stack(parts).sum())
    elif p == 1.0:
        norm = scale * torch.stack([g.double().abs().sum() for g in state["grads"]]).sum()
    else:
        norm = scale * torch.stack([g.abs().max().double() for g in state["grads"]]).max()
    if kind == "grad_norm":
        return norm.float()
    factor = (scale * torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)).float()
    for g in state["grads"]:
        g.copy_(g.float() * factor)
    return {"norm": norm.float(), "grads": dict(state["flat"])}


def run(state):
    if not own:
        return _plain(state)
    case, kind = state["case"], state["case"]["kind"]
    if kind == "norm":
        from pet_kokkos_amd import layer
        layer.norm_rows(state["out"], state["inp"], state["weight"], state["bias"])
        return state["out"]
    if kind == "norm_grads":
        from pet_kokkos_amd import layer
        layer.norm_rows_grads(state["out"], state["w_adj"], state["b_adj"], state["out_adj"], state["inp"],
                              state["weight"], case["ln"], live=state["live"])
        got = {"in_adj": state["out"], "w_adj": state["w_adj"]}
        if case["ln"]:
            got["b_adj"] = state["b_adj"]
        return got
    if kind == "linear_grads":
        from pet_kokkos_amd import linear
        linear.linear_grads(state["out_adj"], state["inp"], state["w_adj"], state["b_adj"], live=state["live"])
        return {"w_adj": state["w_adj"], "b_adj": state["b_adj"]}
    from pet_kokkos_amd import grads
    if kind == "grad_norm":
        return grads.grad_norm(state["list"], norm_type=case["p"], scale=case["scale"])
    norm = grads.clip_grads(state["list"], MAX_NORM, norm_type=case["p"], scale=case["scale"])
    return {"norm": norm, "grads": dict(state["flat"])}


# ---- the work and the definition ----------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_grads"):
        live, width = case.get("live") or case["rows"], case["width"]
        size, vectors = (4 if case["dtype"] == "fp32" else 2), (2 if case["ln"] else 1)
        if kind == "norm":
            return {"bytes": 2 * live * width * size + 4 * vectors * width, "flops": 6 * live * width}
        return {"bytes": 3 * live * width * size + 4 * (1 + vectors) * width, "flops": 16 * live * width}
    if kind == "linear_grads":
        live, n, k = case["live"] or case["rows"], case["n"], case["k"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": live * (n + k) * size + 4 * (n * k + n), "flops": 2 * live * n * k + live * n}
    total = count = 0
    for i, shape in enumerate(_parameter_shapes(case)):
        count += math.prod(shape)
        total += math.prod(shape) * (4 if _grad_dtype(case, i, shape) == "fp32" else 2)
    if kind == "grad_norm":
        return {"bytes": total + 4, "flops": 2 * count}
    return {"bytes": 2 * total + 4, "flops": 3 * count}


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind in ("grad_norm", "clip"):
        total = torch.zeros((), dtype=torch.float64, device=_device())
        for g in state["grads"]:
            a = g.double().abs().flatten()
            if case["p"] == math.inf:
                total = torch.maximum(total, a.max())
            elif case["p"] == 2.0:
                total += torch.dot(a, a)
            else:
                total += a.sum()
        norm = case["scale"] * (total.sqrt() if case["p"] == 2.0 else total)
        if kind == "grad_norm":
            return norm
        factor = case["scale"] * min(1.0, MAX_NORM / (float(norm) + 1e-6))
        return {"norm": norm, "grads": {k: factor * g.double() for k, g in state["flat"].items()}}
    live = case.get("live") or case["rows"]
    if kind == "linear_grads":
        w = torch.zeros((case["n"], case["k"]), dtype=torch.float64, device=_device())
        b = torch.zeros(case["n"], dtype=torch.float64, device=_device())
        for r in range(0, live, 65536):
            g = state["out_adj"][r:min(live, r + 65536)].double()
            w += torch.mm(g.t().contiguous(), state["inp"][r:min(live, r + 65536)].double())
            b += g.sum(0)
        return {"w_adj": w, "b_adj": b}
    width = case["width"]
    weight = state["weight"].double()
    res = torch.zeros((case["rows"], width), dtype=torch.float64, device=_device())
    w = torch.zeros(width, dtype=torch.float64, device=_device())
    b = torch.zeros(width, dtype=torch.float64, device=_device())
    step = max(1, (1 << 25) // width)
    for r in range(0, live, step):
        rows = slice(r, min(live, r + step))
        x = state["inp"][rows].double()
        mean = x.sum(1, keepdim=True) / width if case["ln"] else 0.0
        sd = (((x - mean) ** 2).sum(1, keepdim=True) / width + (LN_EPS if case["ln"] else RMS_EPS)) ** 0.5
        z = (x - mean) / sd
        if kind == "norm":
            res[rows] = z * weight + (state["bias"].double() if case["ln"] else 0.0)
            continue
        g = state["out_adj"][rows].double()
        w += (g * z).sum(0)
        b += g.sum(0)
        h = g * weight
        shift = h.sum(1, keepdim=True) / width if case["ln"] else 0.0
        res[rows] = (h - shift - z * ((h * z).sum(1, keepdim=True) / width)) / sd
    if kind == "norm":
        return res
    got = {"in_adj": res, "w_adj": w}
    if case["ln"]:
        got["b_adj"] = b
    return got
