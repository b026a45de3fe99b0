"""float64 oracle of the operators beside attention: the bias by distance, layer norm, channel mixing
by degree, the gated activation and the 8-bit form of activations.  Plain numpy, written from the
definitions; the gradients by formula (checked against differences in the tests)."""
import numpy as np

from .block import DEGREE


def distance_bias(lengths, boundaries, table, cutoff=None, g=None):
    """bias [E, H]; with g also (grad_table, grad_lengths)."""
    r, table = np.asarray(lengths, np.float64), np.asarray(table, np.float64)
    k = (np.asarray(boundaries, np.float64)[None, :] <= r[:, None]).sum(1)
    out = table[k]
    slope = np.zeros_like(r)
    if cutoff is not None:
        inside = np.abs(r) < cutoff
        u = np.where(inside, r, 0.0) / cutoff
        # 1 - u^2 by factors: no digits are lost next to 1
        out = out + np.where(inside, np.log1p(-u) + np.log1p(u), -np.inf)[:, None]
        slope = np.where(inside, -2 * u / ((1 - u) * (1 + u)) / cutoff, 0.0)
    out = np.where(np.isnan(r)[:, None], np.nan, out)
    if g is None:
        return out
    g = np.asarray(g, np.float64)
    gt = np.zeros_like(table)
    np.add.at(gt, k, g)
    return out, gt, np.where(np.isnan(r), np.nan, slope) * g.sum(1)


def layer_norm(x, weight, bias=None, eps=1e-5, g=None):
    """y; with g also (grad_x, grad_weight, grad_bias); x [R, D]."""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    d = x - x.mean(1, keepdims=True)
    r = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    xh = d * r
    y = xh * weight + (0 if bias is None else np.asarray(bias, np.float64))
    if g is None:
        return y
    g = np.asarray(g, np.float64)
    u = g * weight
    gx = r * (u - u.mean(1, keepdims=True) - xh * (u * xh).mean(1, keepdims=True))
    return y, gx, (g * xh).sum(0), g.sum(0)


def channel_mixing(x, weight, g=None, kept_x=None):
    """y; with g also (grad_x, grad_weight), the latter at kept_x (None: x)."""
    x, w = np.asarray(x, np.float64), np.asarray(weight, np.float64)[DEGREE]      # [16, C, O]
    y = np.einsum("ncm,mco->nom", x, w, optimize=True)
    if g is None:
        return y
    g = np.asarray(g, np.float64)
    gx = np.einsum("nom,mco->ncm", g, w, optimize=True)
    xw = x if kept_x is None else np.asarray(kept_x, np.float64)
    per = np.einsum("ncm,nom->mco", xw, g, optimize=True)
    return y, gx, np.stack([per[DEGREE == l].sum(0) for l in range(4)])


def gate_activation(x, g=None, kept_x=None):
    """y; with g also grad_x, at kept_x (None: x)."""
    x = np.asarray(x, np.float64)

    def on(t):
        t = t[:, :, :1]
        e = np.exp(-np.abs(t))
        return np.where(t >= 0, 1.0, e) / (1 + e), np.where(t >= 0, e, 1.0) / (1 + e)

    y = on(x)[0] * x
    if g is None:
        return y
    g = np.asarray(g, np.float64)
    xk = x if kept_x is None else np.asarray(kept_x, np.float64)
    s, off = on(xk)
    gx = s * g
    gx[:, :, :1] += s * off * (g * xk).sum(2, keepdims=True)
    return y, gx


def e4m3_values():
    """The 127 values of codes 0 to 126 (127 is NaN), by the format's definition."""
    v = []
    for code in range(127):
        e, m = code >> 3, code & 7
        v.append(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return np.array(v)


def encode(x):
    """(codes uint8 [N, C, 16], exponents + 127 uint8 [N, ceil(C / 8)]) of x [N, C, 16]."""
    x = np.asarray(x, np.float64)
    n, c = x.shape[:2]
    values = e4m3_values()
    codes = np.zeros(x.shape, np.uint8)
    exps = np.zeros((n, -(-c // 8)), np.uint8)
    for i in range(n):
        for b in range(exps.shape[1]):
            block = x[i, 8 * b:8 * b + 8]
            top = max([0.0] + [abs(v) for v in block.ravel() if np.isfinite(v)])
            e = -110
            while e < 120 and top > 448 * 2.0 ** e:
                e += 1
            exps[i, b] = e + 127
            q = np.abs(np.where(np.isfinite(block), block, 0)) / 2.0 ** e
            hi = np.clip(np.searchsorted(values, q), 0, 126)
            lo = np.maximum(hi - 1, 0)
            up = values[hi] - q
            down = q - values[lo]
            code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
            if e == 120:
                code = np.minimum(code, 119)        # 240: 256 * 2^120 is no fp32 number
            code = np.where(np.isfinite(block), code, 127)
            codes[i, 8 * b:8 * b + 8] = code | (np.signbit(block).astype(np.uint8) << 7)
    return codes, exps


def decode(codes, exps):
    values = np.append(e4m3_values(), np.nan)
    v = values[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    return v * np.repeat(2.0 ** (exps.astype(np.float64) - 127), 8, 1)[:, :codes.shape[1], None]


def kept(x):
    return decode(*encode(x))
