"""What a user of this package has its training and serving operators do, as measured cases: the
parts of an equivariant transformer that stand beside attention over neighbours.

Four kinds:

  bias      the learned bias of attention by distance buckets, with a smooth cutoff; forward, or with
            the gradients of the table and of the lengths
  layernorm layer norm of rows: hidden features of edges, or an atom's invariants, which lie 16 apart
            in features [N, C, 16]; forward or a training step
  mixing    channels mixed degree by degree (the linear layer of equivariant features); forward, or a
            training step, the layer's input kept for it as it is or in 8 bits
  gate      the gated activation of a feed-forward layer; forward, or a training step, its input kept
            as it is or in 8 bits

Kept in 8 bits ("e4m3"): blocks of 8 channels x 16 components of an atom share a power of two, the
least 2^E with max |x| <= 448 * 2^E (E within [-110, 120]), and hold x / 2^E as e4m3, rounded to nearest
even.  The gradients that need the input are those of the values so kept.
"""
import math
import os
import sys

import torch

own = False

CUTOFF = 5.0
NEIGHBORS = 28          # edges of an atom on average, as in a box of 30 neighbours within the cutoff
EPS = 1e-5
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _bias(atoms, buckets, heads, cutoff, train):
    return {"kind": "bias", "atoms": atoms, "buckets": buckets, "heads": heads, "cutoff": cutoff,
            "dtype": "f32", "train": train}


def _layernorm(rows, size, scalars, dtype, train):
    return {"kind": "layernorm", "rows": rows, "size": size, "scalars": scalars, "dtype": dtype,
            "train": train}


def _mixing(atoms, c_in, c_out, dtype, train, kept):
    return {"kind": "mixing", "atoms": atoms, "c_in": c_in, "c_out": c_out, "dtype": dtype,
            "train": train, "kept": kept}


def _gate(atoms, channels, dtype, train, kept):
    return {"kind": "gate", "atoms": atoms, "channels": channels, "dtype": dtype, "train": train,
            "kept": kept}


def listed():
    return [
        # the edges of one molecule in a serving loop: the smallest call
        dict(_bias(100, 32, 4, True, False), name="bias_100"),
        # a training step of a 5000-atom system's bias, 8 heads
        dict(_bias(5000, 64, 8, True, True), name="bias_5000_train"),
        # the same of 50,000 atoms with fine buckets
        dict(_bias(50000, 256, 8, True, True), name="bias_50000_train"),
        # the invariants of a small system, read where they lie among the components
        dict(_layernorm(1000, 32, True, "f32", False), name="layernorm_1000_32"),
        # hidden features of the edges of 20,011 atoms in a radial network, training in bf16
        dict(_layernorm(20011 * NEIGHBORS, 64, False, "bf16", True),
             name="layernorm_560308_64_bf16_train"),
        # the invariants of a large system, a size that fills no vector, training
        dict(_layernorm(20011, 100, True, "f32", True), name="layernorm_20011_100_train"),
        # the mixing of one molecule in a serving loop
        dict(_mixing(100, 64, 64, "f32", False, ""), name="mixing_100_64"),
        # a training step of a 5000-atom layer, f32
        dict(_mixing(5000, 64, 64, "f32", True, ""), name="mixing_5000_64_train"),
        # a training step of a large system in bf16, the input kept in 8 bits
        dict(_mixing(50000, 128, 128, "bf16", True, "e4m3"),
             name="mixing_50000_128_bf16_e4m3_train"),
        # f32, channels that fill no tile, a wider output, the input kept in 8 bits
        dict(_mixing(20011, 100, 200, "f32", True, "e4m3"), name="mixing_20011_100_e4m3_train"),
        # the activation of a small system's feed-forward layer
        dict(_gate(1000, 64, "f32", False, ""), name="gate_1000_64"),
        # that of a large one's hidden channels, training in bf16, the input kept in 8 bits
        dict(_gate(50000, 256, "bf16", True, "e4m3"), name="gate_50000_256_bf16_e4m3_train"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng, lo, hi):
    """Half of them multiples of 8."""
    c = _log_int(rng, lo, hi)
    return c if rng.random() < 0.5 else max(8, c // 8 * 8)


def draw(rng):
    kind = rng.choice(["bias"] * 3 + ["layernorm"] * 3 + ["mixing"] * 5 + ["gate"] * 2)
    dtype = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.6
    kept = rng.choice(["", "e4m3"]) if train else ""
    most = 50000 * 128
    if kind == "bias":
        return _bias(_log_int(rng, 30, 50000), _log_int(rng, 2, 512), rng.randint(1, 16),
                     rng.random() < 0.7, train)
    if kind == "layernorm":
        size = _channels(rng, 4, 4096)
        if rng.random() < 0.4:
            size = min(size, 256)
            return _layernorm(_log_int(rng, 30, most // max(size, 128)), size, True, dtype, train)
        return _layernorm(_log_int(rng, 30, 50_000_000 // max(size, 32)), size, False, dtype, train)
    if kind == "mixing":
        a, b = _channels(rng, 4, 256), _channels(rng, 4, 256)
        limit = min(50000, most // max(a, b), most * 128 // (a * b))
        return _mixing(_log_int(rng, 30, limit), a, b, dtype, train, kept)
    c = _channels(rng, 4, 512)
    return _gate(_log_int(rng, 30, min(50000, most // c)), c, dtype, train, kept)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _inputs(case, seed):
    """The tensors alone, from the seed."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    t = TYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "bias":
        e, h, b = case["atoms"] * NEIGHBORS, case["heads"], case["buckets"]
        # pairs of uniform density within the cutoff, and each in both directions elsewhere in the list
        r = CUTOFF * torch.rand(e // 2, generator=g, device=DEV) ** (1.0 / 3.0)
        s["lengths"] = torch.cat([r, r.roll(1)])
        s["boundaries"] = torch.arange(1, b, device=DEV) * (CUTOFF / b)
        s["table"] = 0.5 * _randn(g, b, h)
        if case["train"]:
            # attention's gradients: small for most edges, of either sign
            s["g"] = 0.05 * _randn(g, e, h) * torch.rand(e, 1, generator=g, device=DEV)
    elif kind == "layernorm":
        n, d = case["rows"], case["size"]
        if case["scalars"]:
            s["features"] = 0.7 * _randn(g, n, d, 16, dtype=t) + 0.5
            s["x"] = s["features"][:, :, 0]
        else:
            s["x"] = 0.7 * _randn(g, n, d, dtype=t) + 0.5
        s["weight"], s["bias"] = 1 + 0.1 * _randn(g, d), 0.1 * _randn(g, d)
        if case["train"]:
            s["g"] = _randn(g, n, d, dtype=t)
    else:
        n = case["atoms"]
        c = case["c_in"] if kind == "mixing" else case["channels"]
        # each degree and atom of a scale of its own
        scale = torch.tensor([1.0] + [0.7] * 3 + [0.5] * 5 + [0.3] * 7, device=DEV)
        s["x"] = (_randn(g, n, c, 16) * scale
                  * torch.exp(0.5 * _randn(g, n, 1, 1))).to(t)
        if kind == "mixing":
            s["weight"] = _randn(g, 4, c, case["c_out"]) / math.sqrt(c)
        if case["train"]:
            s["g"] = _randn(g, n, case["c_out"] if kind == "mixing" else c, 16, dtype=t)
    return s


_WANTED = {"bias": ("table", "lengths"), "layernorm": ("x", "weight", "bias"),
           "mixing": ("x", "weight"), "gate": ("x",)}


def _wanted(case):
    # without a cutoff the bias is a step function of the lengths, whose gradient is 0
    names = _WANTED[case["kind"]]
    return names[:1] if case["kind"] == "bias" and not case["cutoff"] else names


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        sys.path.insert(0, os.path.abspath(os.path.join("batmobile-evo_amd", "python")))
        import batmobile

        s["batmobile"] = batmobile
        if case["train"]:
            for name in _wanted(case):
                s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"bias": _plain_bias, "layernorm": _plain_layernorm, "mixing": _plain_mixing,
                "gate": _plain_gate}[s["case"]["kind"]](s)


def _own(s):
    case, bm = s["case"], s["batmobile"]
    if case["kind"] == "bias":
        out = bm.distance_bias(s["lengths"], s["boundaries"], s["table"],
                               CUTOFF if case["cutoff"] else None)
    elif case["kind"] == "layernorm":
        out = bm.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    elif case["kind"] == "mixing":
        out = bm.channel_mixing(s["x"], s["weight"], case["kept"] or None)
    else:
        out = bm.gate_activation(s["x"], case["kept"] or None)
    if not case["train"]:
        return {"out": out}
    names = _wanted(case)
    grads = torch.autograd.grad(out, [s[x] for x in names], s["g"])
    return {"out": out, **{"g" + x: t for x, t in zip(names, grads)}}


def _plain_bias(s):
    case, r = s["case"], s["lengths"]
    k = torch.bucketize(r, s["boundaries"], right=True)
    out = s["table"][k]
    if case["cutoff"]:
        # (c - r) (c + r) keeps its precision next to the cutoff
        wide = (CUTOFF - r) * (CUTOFF + r)
        out = out + torch.log((wide / CUTOFF ** 2).clamp(min=0))[:, None]
    if not case["train"]:
        return {"out": out}
    # 256 sums of each bucket, which are shorter and wait less for each other than one, joined in 64 bits
    b, h = s["table"].shape
    slot = torch.arange(k.numel(), device=DEV) % 256
    total = torch.zeros(256 * b, h, device=DEV).index_add_(0, slot * b + k, s["g"])
    res = {"out": out, "gtable": total.view(256, b, h).double().sum(0).float()}
    if case["cutoff"]:
        slope = torch.where(r < CUTOFF, -2 * r / torch.where(r < CUTOFF, wide, 1.0), 0.0)
        res["glengths"] = s["g"].sum(1) * slope
    return res


def _plain_layernorm(s):
    t = s["x"].dtype
    x = s["x"].float()
    x = x - x.mean(1, keepdim=True)
    rs = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
    xh = x * rs
    out = (xh * s["weight"] + s["bias"]).to(t)
    if not s["case"]["train"]:
        return {"out": out}
    g = s["g"].float()
    gw = g * s["weight"]
    gx = rs * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return {"out": out, "gx": gx.to(t), "gweight": (g * xh).sum(0), "gbias": g.sum(0)}


def _plain_kept(x):
    """float32 values of x [N, C, 16] as 8 bits hold them, a power of two for each 8 channels."""
    n, c = x.shape[:2]
    blocks = torch.nn.functional.pad(x.float(), (0, 0, 0, -c % 8)).view(n, -1, 128)
    m, e = torch.frexp(blocks.abs().amax(2, keepdim=True))        # max = m 2^e, 448 = 0.875 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(m == 0, -110, e).clamp(-110, 120)
    up = ((e + 127) << 23).view(torch.float32)                    # 2^e and 2^-e, exactly
    down = ((127 - e) << 23).view(torch.float32)
    return ((blocks * down).to(torch.float8_e4m3fn).float() * up).view(n, -1, 16)[:, :c]


def _plain_mixing(s):
    """Component by component: rows of the atoms times the weight of the component's degree."""
    case = s["case"]
    t = s["x"].dtype
    degree = torch.tensor([0] + [1] * 3 + [2] * 5 + [3] * 7, device=DEV)
    w = s["weight"][degree]                                       # [16, C_in, C_out]
    out = torch.bmm(s["x"].float().permute(2, 0, 1).contiguous(), w)
    res = {"out": out.permute(1, 2, 0).contiguous().to(t)}
    if case["train"]:
        x = _plain_kept(s["x"]) if case["kept"] else s["x"].float()
        g = s["g"].float().permute(2, 0, 1).contiguous()          # [16, N, C_out]
        gx = torch.bmm(g, w.transpose(1, 2).contiguous())
        gw = torch.bmm(x.permute(2, 1, 0).contiguous(), g)
        res["gx"] = gx.permute(1, 2, 0).contiguous().to(t)
        res["gweight"] = torch.zeros_like(s["weight"]).index_add_(0, degree, gw)
    return res


def _plain_gate(s):
    case = s["case"]
    t = s["x"].dtype
    x = s["x"].float()
    res = {"out": (x / (1 + torch.exp(-x[:, :, :1]))).to(t)}
    if case["train"]:
        if case["kept"]:
            x = _plain_kept(s["x"])
        g = s["g"].float()
        on = 1 / (1 + torch.exp(-x[:, :, :1]))
        off = 1 / (1 + torch.exp(x[:, :, :1]))
        gx = on * g
        gx[:, :, :1] += on * off * (g * x).sum(2, keepdim=True)
        res["gx"] = gx.to(t)
    return res


# ---------------------------------------------------------------------------
# the least work of one pass
# ---------------------------------------------------------------------------

def work(case):
    """Each input read once and each output written once; in training the output's gradient is an
    input and the others are outputs."""
    size, train = (2 if case["dtype"] == "bf16" else 4), case["train"]
    if case["kind"] == "bias":
        e, h, table = case["atoms"] * NEIGHBORS, case["heads"], case["buckets"] * case["heads"]
        b, f = 4 * (e + table + e * h), 4 * e + e * h
        if train:
            b += 4 * (table + e * h) + (4 * e if case["cutoff"] else 0)
            f += (2 if case["cutoff"] else 1) * e * h
    elif case["kind"] == "layernorm":
        cells = case["rows"] * case["size"]
        b, f = 2 * size * cells + 8 * case["size"], 8 * cells
        if train:
            b, f = b + 2 * size * cells + 8 * case["size"], f + 14 * cells
    elif case["kind"] == "mixing":
        a, o, w = case["atoms"] * case["c_in"], case["atoms"] * case["c_out"], \
            case["c_in"] * case["c_out"]
        b, f = 16 * size * (a + o) + 16 * w, 32 * case["atoms"] * w
        if train:
            b, f = 2 * b, 3 * f
    else:
        cells = 16 * case["atoms"] * case["channels"]
        b, f = 2 * size * cells, 2 * cells
        if train:
            b, f = 2 * b, f + 4 * cells
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------

def exact(case, seed):
    """The definitions in 64 bits; the gradients by differentiating them."""
    s = _inputs(case, seed)
    names = _wanted(case)
    d = {x: s[x].double().requires_grad_(case["train"]) for x in names}
    kind = case["kind"]
    with torch.enable_grad():
        if kind == "bias":
            r = d.get("lengths", s["lengths"].double())
            out = d["table"][(r[:, None] >= s["boundaries"].double()).sum(1)] \
                if r.numel() * case["buckets"] < 1 << 28 else \
                d["table"][torch.searchsorted(s["boundaries"].double(), r.detach(), side="right")]
            if case["cutoff"]:
                # the derivative at an edge of the cutoff's own length is 0, not that of log 0
                there = r < CUTOFF
                inside = 1 - (torch.where(there, r, 0.0) / CUTOFF) ** 2
                out = out + torch.where(there, inside.log(), -math.inf)[:, None]
        elif kind == "layernorm":
            x = d["x"]
            mean = x.sum(1, keepdim=True) / case["size"]
            var = ((x - mean) ** 2).sum(1, keepdim=True) / case["size"]
            out = (x - mean) / (var + EPS).sqrt() * d["weight"] + d["bias"]
        elif kind == "mixing":
            out = _exact_mixing(d["x"], d["weight"])
        else:
            out = d["x"] * torch.sigmoid(d["x"][:, :, :1])
        if not case["train"]:
            return {"out": out}
        if not case.get("kept"):
            grads = torch.autograd.grad(out, [d[x] for x in names], s["g"].double())
        elif kind == "mixing":
            # the input's gradient needs no input; the weight's is that at the kept input
            gx, = torch.autograd.grad(out, [d["x"]], s["g"].double())
            again = _exact_mixing(_exact_kept(s["x"]), d["weight"])
            grads = gx, *torch.autograd.grad(again, [d["weight"]], s["g"].double())
        else:
            x = _exact_kept(s["x"]).requires_grad_(True)
            grads = torch.autograd.grad(x * torch.sigmoid(x[:, :, :1]), [x], s["g"].double())
    return {"out": out.detach(), **{"g" + x: t for x, t in zip(names, grads)}}


def _exact_mixing(x, weight):
    parts = []
    for l in range(4):
        part = x[:, :, l * l:(l + 1) ** 2].transpose(1, 2)         # [N, 2l + 1, C]
        parts.append(torch.matmul(part.reshape(-1, x.shape[1]), weight[l])
                     .view(x.shape[0], 2 * l + 1, -1))
    return torch.cat(parts, 1).transpose(1, 2)


def _power(e):
    """2^e, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_kept(x):
    """From the definition: steps of 2^-3 of a value's power of two, of 2^-9 at the least."""
    x = x.double()
    out = torch.empty_like(x)
    for a in range(0, x.shape[1], 8):
        block = x[:, a:a + 8]
        top = block.abs().amax((1, 2), keepdim=True)
        e = torch.ceil(torch.log2(top / 448).clamp(-110, 120))
        # log2 rounds: the least power is the one that holds, whose half does not
        e = torch.where((448 * _power(e - 1) >= top) & (e > -110), e - 1, e)
        e = torch.where((448 * _power(e) < top) & (e < 120), e + 1, e)
        unit = _power(e)
        v = block / unit
        step = _power((torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
        out[:, a:a + 8] = torch.round(v / step) * step * unit
    return out
