"""float64 oracle of the operators of an equivariant transformer block: attention over the edges
of a graph, norms by degree with gate and residual, gradient clipping.  Plain numpy, written from
the definitions; the gradients by formula (checked against differences in the tests)."""
import numpy as np

DEGREE = np.array([0] + [1] * 3 + [2] * 5 + [3] * 7)


def attention(q, k, v, src, row_ptr, bias=None, scale=None, go=None):
    """(out, grads): rows in row_ptr order, src the sources; an edge whose bias or logit is -inf
    does not exist.  With go: {"q", "k", "v", "bias"}."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    n, h, dk = q.shape
    group = h // k.shape[1]
    scale = dk ** -0.5 if scale is None else scale
    out = np.zeros((n, h, v.shape[2]))
    g = {"q": np.zeros_like(q), "k": np.zeros_like(k), "v": np.zeros_like(v),
         "bias": np.zeros((len(src), h))}
    for i in range(n):
        e0, e1 = int(row_ptr[i]), int(row_ptr[i + 1])
        for hh in range(h):
            j, kv = np.asarray(src[e0:e1], np.int64), hh // group
            b = np.zeros(e1 - e0) if bias is None else np.asarray(bias[e0:e1, hh], np.float64)
            on = b > -np.inf
            on[np.isnan(b)] = True
            e, j, b = np.arange(e0, e1)[on], j[on], b[on]
            if not len(e):
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                x = scale * (k[j, kv] @ q[i, hh]) + b
                keep = ~(x == -np.inf)
                e, j, x = e[keep], j[keep], x[keep]
                if not len(e):
                    continue
                p = np.exp(x - x.max())
                p = p / p.sum()
                out[i, hh] = p @ v[j, kv]
                if go is not None:
                    w = np.asarray(go[i, hh], np.float64)
                    dp = v[j, kv] @ w
                    ds = p * (dp - p @ dp)
                    g["bias"][e, hh] = ds
                    g["q"][i, hh] = scale * (ds @ k[j, kv])
                    np.add.at(g["k"][:, kv], j, scale * ds[:, None] * q[i, hh])
                    np.add.at(g["v"][:, kv], j, p[:, None] * w)
    return (out, g) if go is not None else out


def norm(z, w, eps=1e-6):
    """(norm(z; w), 1 / rms by degree [N, 4])."""
    z = np.asarray(z, np.float64)
    r = np.stack([1 / np.sqrt((z[:, :, DEGREE == l] ** 2).mean((1, 2)) + eps) for l in range(4)], 1)
    return z * r[:, None, DEGREE] * np.asarray(w, np.float64).T[None][:, :, DEGREE], r


def _norm_grad(z, r, w, g):
    w = np.asarray(w, np.float64).T[:, DEGREE]
    back, gw = np.zeros_like(z), np.zeros((4, z.shape[1]))
    for l in range(4):
        on = DEGREE == l
        rl = r[:, l][:, None, None]
        dot = (g[:, :, on] * w[:, on] * z[:, :, on]).mean((1, 2), keepdims=True)
        back[:, :, on] = rl * w[:, on] * g[:, :, on] - rl ** 3 * dot * z[:, :, on]
        gw[l] = (g[:, :, on] * z[:, :, on] * rl).sum((0, 2))
    return back, gw


def gated_residual_norm(x, y, gate, scale, w_post, w_pre, eps=1e-6, gh=None, gn=None):
    """(h, n[, grads]); y None: (x, norm(x)); gate None: factor 1; w_pre None: n is None."""
    x = np.asarray(x, np.float64)
    train = gh is not None or gn is not None
    g = {}
    h = x
    if y is not None:
        y = np.asarray(y, np.float64)
        s = 1 / (1 + np.exp(-np.asarray(gate, np.float64))) if gate is not None \
            else np.ones(x.shape[:2] + (4,))
        # 1 - s, where s is next to 1 as well
        off = 1 / (1 + np.exp(np.asarray(gate, np.float64))) if gate is not None else 0
        sc = np.asarray(scale, np.float64)[None, :, None]
        post, ry = norm(y, w_post, eps)
        h = x + sc * s[:, :, DEGREE] * post
    n, rh = norm(h, w_pre, eps) if w_pre is not None else (None, None)
    if not train:
        return h, n
    G = np.zeros_like(h) if gh is None else np.asarray(gh, np.float64)
    if gn is not None:
        back, g["w_pre"] = _norm_grad(h, rh, w_pre, np.asarray(gn, np.float64))
        G = G + back
    g["x"] = G
    if y is not None:
        g["y"], g["w_post"] = _norm_grad(y, ry, w_post, G * sc * s[:, :, DEGREE])
        by = np.stack([(G * post)[:, :, DEGREE == l].sum(2) for l in range(4)], 2)
        g["gate"] = by * sc * s * off
        g["scale"] = (by * s).sum((0, 2))
    return h, n, g


def clip(grads, max_norm):
    """(norm, clipped)."""
    grads = [np.asarray(t, np.float64) for t in grads]
    norm = np.sqrt(sum((t ** 2).sum() for t in grads))
    with np.errstate(invalid="ignore", divide="ignore"):
        r = max_norm / (norm + 1e-6)
        c = r if not r >= 1.0 else 1.0
        return norm, [t * c for t in grads]
