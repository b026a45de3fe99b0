"""What a user of this package has its training and serving operators do, as measured cases.

Three kinds, the parts of an equivariant transformer's step that stand beside the message
passing kernels:

  attention   softmax attention of every destination over its incoming edges (shared key/value
              heads, a bias per edge and head), forward or a training step
  norm        normalisation of features [N, C, 16] by degree: alone ("pre"), or of a block's
              output with its gate, residual scale and the next block's norm ("block"), forward
              or a training step
  clip        global norm of many gradient tensors, and the clipped gradients

Graphs: "box", atoms of a periodic cube, every pair up to the length that gives 28 neighbours on
average; "random", the caller's own edge list in no order, sources uniform; "readout", a few query rows per system
that attend to every atom of it.
"""
import math
import os
import sys

import torch

own = False

CUTOFF = 5.0
DENSITY = 30.0 / (4.0 / 3.0 * math.pi * CUTOFF ** 3)
NEIGHBORS = 28          # of an atom of a box on average: the edge count is the same for all seeds
EPS = 1e-6
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
DEGREE = [0] + [1] * 3 + [2] * 5 + [3] * 7   # degree l of each of the 16 components


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _attention(graph, atoms, heads, kv_heads, dk, dv, dtype, train, rows=0, systems=0):
    return {"kind": "attention", "graph": graph, "atoms": atoms, "heads": heads,
            "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype, "train": train,
            "rows": rows, "systems": systems}


def _norm(form, atoms, channels, dtype, train):
    return {"kind": "norm", "form": form, "atoms": atoms, "channels": channels, "dtype": dtype,
            "train": train}


def _clip(layers, channels, dtype, max_norm):
    return {"kind": "clip", "layers": layers, "channels": channels, "dtype": dtype,
            "max_norm": max_norm}


def listed():
    return [
        # one molecule in a serving loop: the smallest call, where launches count
        dict(_attention("box", 100, 4, 4, 128, 128, "f32", False), name="attention_100"),
        # one layer of a 5000-atom system with 64 channels in 8 heads of 8 x 16 components
        dict(_attention("box", 5000, 8, 8, 128, 128, "f32", False), name="attention_5000"),
        # the same layer of 50,000 atoms and 128 channels, bf16
        dict(_attention("box", 50000, 8, 8, 256, 256, "bf16", False),
             name="attention_50000_bf16"),
        # four readout queries over the atoms of each of two systems: few rows, long ones
        dict(_attention("readout", 50001, 4, 4, 64, 128, "bf16", False, rows=4, systems=2),
             name="readout_50001_bf16"),
        # a training step of the 5000-atom layer
        dict(_attention("box", 5000, 8, 8, 128, 128, "f32", True), name="attention_5000_train"),
        # a training step in bf16, two key/value heads for eight query heads, an odd atom count
        dict(_attention("box", 20011, 8, 2, 128, 128, "bf16", True),
             name="attention_20011_shared_train"),
        # a training step on the caller's own edge list: invariant keys, sources anywhere
        dict(_attention("random", 5000, 4, 4, 24, 256, "f32", True),
             name="attention_5000_random_train"),
        # the norm before the first block of a small system
        dict(_norm("pre", 1000, 32, "f32", False), name="norm_1000_32"),
        # a block's norm, gate, residual and next norm at scale, inference in bf16
        dict(_norm("block", 50000, 128, "bf16", False), name="norm_block_50000_128_bf16"),
        # the same as a training step, fp32, a channel count that fills no tile
        dict(_norm("block", 20011, 100, "f32", True), name="norm_block_20011_100_train"),
        # the gradients of a two-layer network with shared path weights, clipped
        dict(_clip(2, 32, "f32", 0.5), name="clip_2_32"),
        # those of a large one, mixed types
        dict(_clip(12, 256, "mixed", 10.0), name="clip_12_256_mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention"] * 5 + ["norm"] * 3 + ["clip"] * 2)
    dtype = rng.choice(["f32", "bf16"])
    if kind == "attention":
        most = work(listed()[2])["flops"]
        while True:
            graph = rng.choice(["box", "box", "box", "random", "readout"])
            kv = rng.choice([1, 2, 3, 4, 8])
            heads = kv * rng.choice([1, 1, 2, 4])
            dv = 16 * rng.randint(1, 16) if rng.random() < 0.8 else rng.randint(4, 256)
            dk = dv if rng.random() < 0.6 else rng.randint(4, 128)
            atoms = _log_int(rng, 30, {"box": 50000, "random": 20000, "readout": 100000}[graph])
            rows = rng.randint(1, 8) if graph == "readout" else 0
            systems = rng.randint(1, max(1, min(16, atoms // 8))) if graph == "readout" else 0
            case = _attention(graph, atoms, heads, kv, dk, dv, dtype, rng.random() < 0.5, rows,
                              systems)
            if work(case)["flops"] <= most:
                return case
    if kind == "norm":
        c = _log_int(rng, 4, 256)
        c = c if rng.random() < 0.3 else (c + 7) // 8 * 8
        return _norm(rng.choice(["pre", "block", "block"]),
                     _log_int(rng, 30, 50000 * 128 // max(c, 128)), c, dtype,
                     rng.random() < 0.6)
    return _clip(rng.randint(1, 12), _log_int(rng, 4, 256), rng.choice(["f32", "bf16", "mixed"]),
                 rng.choice([0.01, 1.0, 10.0, 1e6]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _box_graph(g, n):
    """(dst, src, length, positions, cell): the NEIGHBORS * n shortest edges of a periodic cube
    (both directions of a pair), dst then src ascending."""
    side = (n / DENSITY) ** (1.0 / 3.0)
    pos = torch.rand(n, 3, generator=g, device=DEV) * side
    reach = 1.1 * CUTOFF if n > 1000 else 2 * side
    rows = max(1, 50_000_000 // n)
    pairs, square = [], []
    for i0 in range(0, n, rows):
        d2 = torch.zeros(min(rows, n - i0), n, device=DEV)
        for a in range(3):
            t = pos[i0:i0 + rows, None, a] - pos[None, :, a]
            t = t - torch.round(t / side) * side
            d2 += t * t
        # each pair once, the second direction added below
        i = torch.arange(i0, i0 + d2.shape[0], device=DEV)[:, None]
        p = ((d2 <= reach * reach) & (i < torch.arange(n, device=DEV))).nonzero()
        square.append(d2[p[:, 0], p[:, 1]])
        pairs.append(p + torch.tensor([i0, 0], device=DEV))
    pairs, square = torch.cat(pairs), torch.cat(square)
    keep = torch.argsort(square)[:NEIGHBORS * n // 2]
    i, j, d = pairs[keep, 0], pairs[keep, 1], square[keep].sqrt()
    dst, src, d = torch.cat([i, j]), torch.cat([j, i]), torch.cat([d, d])
    by = torch.argsort(dst * n + src)
    return dst[by].contiguous(), src[by].contiguous(), d[by], pos, \
        torch.diag(torch.full((3,), side))


def _random_graph(g, n):
    """(dst, src): 20 to 40 edges per destination, sources uniform, edges in no order."""
    count = (20 + torch.arange(n, device=DEV) % 21)[torch.randperm(n, generator=g, device=DEV)]
    dst = torch.repeat_interleave(torch.arange(n, device=DEV), count)
    src = torch.randint(0, n, (dst.numel(),), generator=g, device=DEV)
    p = torch.randperm(dst.numel(), generator=g, device=DEV)
    return dst[p].contiguous(), src[p].contiguous()


def _readout_graph(g, n, systems, rows):
    """(dst, src): the atoms cut into systems of uneven sizes, `rows` query rows for each."""
    cut = torch.randperm(n - 1, generator=g, device=DEV)[:systems - 1].sort().values + 1
    edge = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), cut,
                      torch.full((1,), n, device=DEV)])
    dst, src = [], []
    for s, (a, b) in enumerate(zip(edge[:-1].tolist(), edge[1:].tolist())):
        for r in range(rows):
            src.append(torch.arange(a, b, device=DEV))
            dst.append(torch.full((b - a,), s * rows + r, device=DEV))
    return torch.cat(dst), torch.cat(src)


def _shapes(case):
    """The parameter tensors of `layers` layers: path weights, radial MLP, norms, projections."""
    c = case["channels"]
    out = []
    for _ in range(case["layers"]):
        out += [(34, c, c), (8, 64), (64,), (64, 34 * c), (4, c), (4, c), (c,), (c, 3 * c),
                (c, c), (4, c, c)]
    return out + [(17, c), (c, 16), (16,), (16, 1), (1,)]


def _inputs(case, seed):
    """The tensors alone, from the seed."""
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "attention":
        t = TYPES[case["dtype"]]
        n, h, kv, dk, dv = (case[x] for x in ("atoms", "heads", "kv_heads", "dk", "dv"))
        if case["graph"] == "box":
            s["dst"], s["src"], dist, s["pos"], s["cell"] = _box_graph(g, n)
            # log of a smooth envelope, -inf at the length of the longest edges
            s["bias"] = torch.log((1 - (dist / dist.max()) ** 2).clamp(min=0))[:, None] + \
                0.5 * _randn(g, dist.numel(), h)
        elif case["graph"] == "random":
            s["dst"], s["src"] = _random_graph(g, n)
            s["bias"] = _randn(g, s["dst"].numel(), h)
        else:
            s["dst"], s["src"] = _readout_graph(g, n, case["systems"], case["rows"])
            s["bias"] = None
        s["n_dst"] = case["systems"] * case["rows"] if case["graph"] == "readout" else n
        s["q"] = _randn(g, s["n_dst"], h, dk, dtype=t)
        s["k"] = _randn(g, n, kv, dk, dtype=t)
        s["v"] = _randn(g, n, kv, dv, dtype=t)
        if case["train"]:
            s["gout"] = _randn(g, s["n_dst"], h, dv, dtype=t)
    elif case["kind"] == "norm":
        t = TYPES[case["dtype"]]
        n, c = case["atoms"], case["channels"]
        s["x"] = _randn(g, n, c, 16, dtype=t)
        s["w_pre"] = 1 + 0.1 * _randn(g, 4, c)
        if case["form"] == "block":
            # a block's raw output: each degree of a scale of its own
            degree = torch.tensor(DEGREE, device=DEV)
            s["y"] = (_randn(g, n, c, 16) * torch.tensor([3.0, 1.0, 0.5, 0.2],
                                                         device=DEV)[degree]).to(t)
            s["gate"] = _randn(g, n, c, 4, dtype=t)
            s["scale"] = 0.1 + 0.02 * _randn(g, c)
            s["w_post"] = 1 + 0.1 * _randn(g, 4, c)
        if case["train"]:
            s["gn"] = _randn(g, n, c, 16, dtype=t)
            if case["form"] == "block":
                s["gh"] = _randn(g, n, c, 16, dtype=t)
    else:
        s["grads"] = []
        for i, shape in enumerate(_shapes(case)):
            bf = case["dtype"] == "bf16" or (case["dtype"] == "mixed" and len(shape) > 1)
            s["grads"].append(_randn(g, *shape, dtype=TYPES["bf16" if bf else "f32"])
                              * 10.0 ** -(i % 4))
        # the clipped gradients go into one flat buffer of each type, where an optimizer reads
        s["flat"] = {t: torch.empty(sum(x.numel() for x in s["grads"] if x.dtype == t),
                                    dtype=t, device=DEV) for t in TYPES.values()}
        s["out"], at = [], dict.fromkeys(s["flat"], 0)
        for x in s["grads"]:
            s["out"].append(s["flat"][x.dtype][at[x.dtype]:at[x.dtype] + x.numel()].view_as(x))
            at[x.dtype] += x.numel()
    return s


def _flat(norm, flat):
    return {"norm": norm, "f32": flat[torch.float32], "bf16": flat[torch.bfloat16]}


_GRADS = {"attention": ("q", "k", "v", "bias"), "pre": ("x", "w_pre"),
          "block": ("x", "y", "gate", "scale", "w_post", "w_pre")}


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    sys.path.insert(0, os.path.abspath(os.path.join("batmobile-evo_amd", "python")))
    import batmobile

    s["batmobile"] = batmobile
    if case["kind"] == "attention":
        n, rows = case["atoms"], s["n_dst"]
        if case["graph"] == "random":
            edges = torch.stack([s["src"], s["dst"]])
            s["plan"] = batmobile.AttentionPlan.from_edge_index(edges, rows, n)
        else:
            row_ptr = torch.zeros(rows + 1, dtype=torch.long, device=DEV)
            row_ptr[1:] = torch.bincount(s["dst"], minlength=rows).cumsum(0)
            order = batmobile.spatial_order(s["pos"], s["cell"]) if "pos" in s else None
            s["plan"] = batmobile.AttentionPlan(s["src"], row_ptr, n, order, order)
        if case["train"]:
            s["plan"].source_side()
    if case.get("train"):
        for name in _GRADS[case.get("form", "attention")]:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attention": _own_attention, "norm": _own_norm, "clip": _own_clip}[kind](s)
    with torch.no_grad():
        return {"attention": _plain_attention, "norm": _plain_norm, "clip": _plain_clip}[kind](s)


def _own_attention(s):
    out = s["batmobile"].neighbor_attention(s["q"], s["k"], s["v"], s["plan"], bias=s["bias"])
    if not s["case"]["train"]:
        return {"out": out}
    names = [x for x in _GRADS["attention"] if s[x] is not None]
    grads = torch.autograd.grad(out, [s[x] for x in names], s["gout"])
    return {"out": out, **{"g" + x: t for x, t in zip(names, grads)}}


def _own_norm(s):
    case, bm = s["case"], s["batmobile"]
    names = _GRADS[case["form"]]
    if case["form"] == "pre":
        n = bm.equivariant_norm(s["x"], s["w_pre"], EPS)
        out, outs, seeds = {"n": n}, [n], [s.get("gn")]
    else:
        h, n = bm.gated_residual_norm(s["x"], s["y"], s["gate"], s["scale"], s["w_post"],
                                      s["w_pre"], EPS)
        out, outs, seeds = {"h": h, "n": n}, [h, n], [s.get("gh"), s.get("gn")]
    if case["train"]:
        grads = torch.autograd.grad(outs, [s[x] for x in names], seeds)
        out.update({"g" + x: t for x, t in zip(names, grads)})
    return out


def _own_clip(s):
    norm, _ = s["batmobile"].clip_grad_norm(s["grads"], s["case"]["max_norm"], s["out"])
    return _flat(norm, s["flat"])


def _plain_attention(s):
    case = s["case"]
    t = TYPES[case["dtype"]]
    dst, src, n = s["dst"], s["src"], s["n_dst"]
    h, kv, dk, dv = (case[x] for x in ("heads", "kv_heads", "dk", "dv"))
    group = h // kv
    scale = 1.0 / math.sqrt(dk)
    q = s["q"].float()
    k = s["k"].float().repeat_interleave(group, 1)
    v = s["v"].float().repeat_interleave(group, 1)
    qe, ke, ve = q[dst], k[src], v[src]
    x = (qe * ke).sum(-1) * scale
    if s["bias"] is not None:
        x = x + s["bias"]
    top = torch.full((n, h), -math.inf, device=DEV).scatter_reduce_(
        0, dst[:, None].expand(-1, h), x, "amax")
    top = torch.where(torch.isinf(top), 0.0, top)
    p = torch.exp(x - top[dst])
    total = torch.zeros(n, h, device=DEV).index_add_(0, dst, p)
    p = p / torch.where(total > 0, total, 1.0)[dst]
    out = torch.zeros(n, h, dv, device=DEV).index_add_(0, dst, p[:, :, None] * ve)
    if not case["train"]:
        return {"out": out.to(t)}
    go = s["gout"].float()
    ge = go[dst]
    ds = p * ((ge * ve).sum(-1) - (go * out).sum(-1)[dst])
    gq = torch.zeros(n, h, dk, device=DEV).index_add_(0, dst, ds[:, :, None] * ke) * scale
    m = case["atoms"]
    gk = torch.zeros(m, h, dk, device=DEV).index_add_(0, src, ds[:, :, None] * qe) * scale
    gv = torch.zeros(m, h, dv, device=DEV).index_add_(0, src, p[:, :, None] * ge)
    res = {"out": out.to(t), "gq": gq.to(t), "gk": gk.view(m, kv, group, dk).sum(2).to(t),
           "gv": gv.view(m, kv, group, dv).sum(2).to(t)}
    if s["bias"] is not None:
        res["gbias"] = ds
    return res


def _plain_rms(x, degree):
    """1 / rms of each degree, spread over the 16 components [N, 1, 16]."""
    cols = []
    for l in range(4):
        cols.append((x[:, :, degree == l].square().mean((1, 2)) + EPS).rsqrt())
    return torch.stack(cols, 1)[:, degree][:, None, :]


def _plain_norm_grad(x, r, w, g, degree):
    """Gradients of n = w r x by x and by w [4, C]."""
    a = g * w.t()[:, degree]
    back = torch.zeros_like(x)
    gw = []
    for l in range(4):
        on = degree == l
        mean = (a[:, :, on] * x[:, :, on]).mean((1, 2))[:, None, None]
        rl = r[:, :, on]
        back[:, :, on] = rl * a[:, :, on] - rl ** 3 * mean * x[:, :, on]
        gw.append((g[:, :, on] * x[:, :, on] * rl).sum((0, 2)))
    return back, torch.stack(gw)


def _plain_norm(s):
    case = s["case"]
    t = TYPES[case["dtype"]]
    degree = torch.tensor(DEGREE, device=DEV)
    x = s["x"].float()
    if case["form"] == "pre":
        r = _plain_rms(x, degree)
        out = {"n": (x * r * s["w_pre"].t()[:, degree]).to(t)}
        if case["train"]:
            gx, gw = _plain_norm_grad(x, r, s["w_pre"], s["gn"].float(), degree)
            out.update(gx=gx.to(t), gw_pre=gw)
        return out
    y = s["y"].float()
    gate = 1.0 / (1.0 + torch.exp(-s["gate"].float()))
    scale = s["scale"][:, None]
    ry = _plain_rms(y, degree)
    post = y * ry * s["w_post"].t()[:, degree]
    h = x + scale * gate[:, :, degree] * post
    rh = _plain_rms(h, degree)
    out = {"h": h.to(t), "n": (h * rh * s["w_pre"].t()[:, degree]).to(t)}
    if case["train"]:
        back, gw_pre = _plain_norm_grad(h, rh, s["w_pre"], s["gn"].float(), degree)
        gh = s["gh"].float() + back
        gp = gh * post
        by_degree = torch.stack([gp[:, :, degree == l].sum(2) for l in range(4)], 2)
        gy, gw_post = _plain_norm_grad(y, ry, s["w_post"], gh * scale * gate[:, :, degree],
                                       degree)
        out.update(gx=gh.to(t), gy=gy.to(t),
                   ggate=(by_degree * scale * gate * (1 - gate)).to(t),
                   gscale=(by_degree * gate).sum((0, 2)), gw_post=gw_post, gw_pre=gw_pre)
    return out


def _plain_clip(s):
    total = torch.zeros((), device=DEV)
    for g in s["grads"]:
        total = total + g.float().square().sum()
    norm = total.sqrt()
    coef = (s["case"]["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, out in zip(s["grads"], s["out"]):
        out.copy_(g.float() * coef)
    return _flat(norm, s["flat"])


# ---------------------------------------------------------------------------
# the least work of one pass
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "clip":
        b = f = 0
        for shape in _shapes(case):
            n = math.prod(shape)
            bf = case["dtype"] == "bf16" or (case["dtype"] == "mixed" and len(shape) > 1)
            b += 2 * n * (2 if bf else 4)
            f += 3 * n
        return {"bytes": b, "flops": f}
    size = 2 if case["dtype"] == "bf16" else 4
    n = case["atoms"]
    if case["kind"] == "norm":
        cells = n * case["channels"] * 16
        block = case["form"] == "block"
        b = cells * size * (4 if block else 2)
        f = cells * (10 if block else 4)
        if block:
            b += n * case["channels"] * 4 * size
        if case["train"]:
            # gradients in (gh, gn / gn) and out (gx, gy, the gate's / gx)
            b += cells * size * (4 if block else 2) + (n * case["channels"] * 4 * size
                                                       if block else 0)
            f += cells * (25 if block else 9)
        return {"bytes": b, "flops": f}
    h, kv, dk, dv = (case[x] for x in ("heads", "kv_heads", "dk", "dv"))
    readout = case["graph"] == "readout"
    rows = case["systems"] * case["rows"] if readout else n
    edges = n * case["rows"] if readout else NEIGHBORS * n
    bias = 0 if readout else 4 * h * edges
    # q, k, v and the edges in, out
    b = size * (rows * h * (dk + dv) + n * kv * (dk + dv)) + bias + 8 * edges
    f = 2 * edges * h * (dk + dv)
    if case["train"]:
        # the gradient in, those of q, k, v and the bias out
        b += size * (rows * h * (dk + dv) + n * kv * (dk + dv)) + bias
        f += 2 * edges * h * (3 * dk + 2 * dv)
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "norm": _exact_norm,
                "clip": _exact_clip}[case["kind"]](s)


def _exact_attention(s):
    """Rows in chunks, the edges of a row laid out as one padded line, a softmax along it."""
    case = s["case"]
    n, m = s["n_dst"], case["atoms"]
    h, kv, dk, dv = (case[x] for x in ("heads", "kv_heads", "dk", "dv"))
    by_row = torch.argsort(s["dst"], stable=True)
    degree = torch.bincount(s["dst"], minlength=n)
    start = degree.cumsum(0) - degree
    width = max(1, int(degree.max()))
    rows = max(1, 120_000_000 // (width * max(dk, dv)))
    z = {"dtype": torch.float64, "device": DEV}
    out, gq = torch.zeros(n, h, dv, **z), torch.zeros(n, h, dk, **z)
    gk, gv = torch.zeros(m, kv, dk, **z), torch.zeros(m, kv, dv, **z)
    gb = torch.zeros(s["dst"].numel(), h, **z)
    for a in range(0, n, rows):
        b = min(n, a + rows)
        col = torch.arange(width, device=DEV)[None, :]
        there = col < degree[a:b, None]
        edge = by_row[(start[a:b, None] + col).clamp(max=max(0, by_row.numel() - 1))]
        at = s["src"][edge]
        for i in range(h):
            j = i // (h // kv)
            q = s["q"][a:b, i].double()[:, None, :]
            k, v = s["k"][:, j].double()[at], s["v"][:, j].double()[at]
            x = (q * k).sum(2) / dk ** 0.5
            if s["bias"] is not None:
                x = x + s["bias"][:, i].double()[edge]
            x = x.masked_fill(~there, -math.inf)
            p = torch.nan_to_num(torch.softmax(x, 1), nan=0.0)[:, :, None]
            out[a:b, i] = (p * v).sum(1)
            if case["train"]:
                go = s["gout"][a:b, i].double()[:, None, :]
                dp = (go * v).sum(2, keepdim=True)
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                gb[edge[there], i] = ds[:, :, 0][there]
                gq[a:b, i] = (ds * k).sum(1) / dk ** 0.5
                gk[:, j].index_add_(0, at[there], (ds * q)[there] / dk ** 0.5)
                gv[:, j].index_add_(0, at[there], (p * go)[there])
    res = {"out": out}
    if case["train"]:
        res.update(gq=gq, gk=gk, gv=gv)
        if s["bias"] is not None:
            res["gbias"] = gb
    return res


def _exact_norm(s):
    """The definition in 64 bits; the gradients by differentiating it."""
    case = s["case"]
    names = _GRADS[case["form"]]
    d = {x: s[x].double().requires_grad_(case["train"]) for x in names}

    def spread(t):
        """[..., 4] by degree -> [..., 16]."""
        return torch.cat([t[..., l:l + 1].expand(*t.shape[:-1], 2 * l + 1) for l in range(4)], -1)

    def norm(x, w):
        parts = [((x[..., l * l:(l + 1) ** 2] ** 2).sum((1, 2)) / (x.shape[1] * (2 * l + 1)) + EPS)
                 ** -0.5 for l in range(4)]
        return x * spread(torch.stack(parts, 1))[:, None] * spread(w.transpose(0, 1))

    with torch.enable_grad():
        if case["form"] == "pre":
            outs, seeds = {"n": norm(d["x"], d["w_pre"])}, ["gn"]
        else:
            h = d["x"] + d["scale"][:, None] * spread(torch.sigmoid(d["gate"])) * \
                norm(d["y"], d["w_post"])
            outs, seeds = {"h": h, "n": norm(h, d["w_pre"])}, ["gh", "gn"]
        if not case["train"]:
            return outs
        grads = torch.autograd.grad(list(outs.values()), [d[x] for x in names],
                                    [s[x].double() for x in seeds])
    return {**{k: t.detach() for k, t in outs.items()},
            **{"g" + x: t for x, t in zip(names, grads)}}


def _exact_clip(s):
    norm = torch.cat([g.double().flatten() for g in s["grads"]]).norm()
    coef = min(1.0, s["case"]["max_norm"] / (float(norm) + 1e-6))
    none = [torch.zeros(0, dtype=torch.float64, device=DEV)]
    return _flat(norm, {t: torch.cat(none + [g.double().flatten() * coef for g in s["grads"]
                                             if g.dtype == t]) for t in TYPES.values()})
