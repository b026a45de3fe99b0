"""The operators beside attention on the GPU against the float64 oracle: bias by distance, layer norm,
channel mixing, gated activation, activations in 8 bits.

Bounds, u = 2^-24 (fp32) the rounding of a result, 2^-8 that of bf16:
  bias        table + log: u of each, and the logarithm of a product of five roundings: 8 u (1 + |log|)
  gtable      a sum of n terms, in any order: (n + 8) u sum |g|
  glengths    the same over the heads, and six roundings of the factor
  layer norm  normwise: sums of up to 8192 terms by lanes (chains of 32 and trees), the root, three
              products: 3e-6 of a row's terms; with bf16 results 2^-8 more
  mixing      every term of a sum of K as exact as an fp32 product, one rounding each: (K + 16) u sum |x w|;
              bf16: the weight to 2^-15 (its leading 8 bits, and 8 of the rest to nearest: 2^-7 2^-8), the
              result to 2^-8 of itself more
  gate        the sigmoid to 8 u, three products: 16 u of the terms' absolute sum
"""
import numpy as np
import pytest
import torch

import _batmobile
from oracle import layers as ol

from helpers import gen, normwise_err

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24
ROUND = {"f32": U, "bf16": 2.0 ** -8}


def _np(t):
    return None if t is None else t.detach().cpu().double().numpy()


def _within(got, want, bound):
    got, want = _np(got), np.asarray(want)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                           float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300))))


# ---------------------------------------------------------------------------
# bias by distance
# ---------------------------------------------------------------------------

def _bias_inputs(e, b, h, seed, cutoff=5.0):
    g = gen(seed)
    r = cutoff * 1.05 * torch.rand(e, generator=g)
    bound = torch.sort(cutoff * torch.rand(b - 1, generator=g)).values
    if e > 4 and b > 1:
        r[0], r[1] = bound[0], torch.nextafter(bound[0], torch.tensor(0.0))
        r[2], r[3] = cutoff, torch.nextafter(torch.tensor(cutoff), torch.tensor(0.0))
    return r, bound, torch.randn(b, h, generator=g), torch.randn(e, h, generator=g)


def _check_bias(dev, e, b, h, cutoff, seed):
    import batmobile
    r, bound, table, g = _bias_inputs(e, b, h, seed)
    rd, td = r.to(dev).requires_grad_(True), table.to(dev).requires_grad_(True)
    out = batmobile.distance_bias(rd, bound.to(dev), td, cutoff)
    gr, gt = torch.autograd.grad(out, [rd, td], g.to(dev))
    want, wt, wr = ol.distance_bias(_np(r), _np(bound), _np(table), cutoff, _np(g))
    got = _np(out)
    lost = np.isneginf(want)
    assert np.array_equal(lost, np.isneginf(got))
    env = want - _np(table)[(_np(bound)[None] <= _np(r)[:, None]).sum(1)]
    keep = ~lost
    assert (np.abs(got - np.where(keep, want, 0))[keep]
            <= (8 * U * (1 + np.abs(env) + np.abs(want)))[keep]).all()
    k = (_np(bound)[None] <= _np(r)[:, None]).sum(1)
    absum, count = np.zeros((b, h)), np.zeros((b, 1))
    np.add.at(absum, k, np.abs(_np(g)))
    np.add.at(count, k, 1)
    _within(gt, wt, (count + 8) * U * absum)
    slope = np.abs(wr) / np.maximum(np.abs(_np(g).sum(1)), 1e-300) if h else 0
    _within(gr, wr, U * (h + 8) * slope * np.abs(_np(g)).sum(1) + 8 * U * np.abs(wr))
    assert torch.equal(batmobile.distance_bias(r.to(dev), bound.to(dev), table.to(dev), cutoff), out)


@pytest.mark.parametrize("e,b,h", [(0, 3, 2), (1, 1, 1), (2, 2, 3), (255, 7, 4), (256, 63, 5),
                                   (257, 64, 8), (1000, 65, 16), (5000, 128, 8), (3001, 129, 3),
                                   (20000, 300, 12), (2000, 4096, 2), (700, 9, 33), (300, 20, 64),
                                   (300, 20, 65), (200, 70, 130), (40, 3, 1024)])
@pytest.mark.parametrize("cutoff", [5.0, None])
def test_distance_bias(dev, e, b, h, cutoff):
    _check_bias(dev, e, b, h, cutoff, e + b + h)


def test_distance_bias_odd_lengths(dev):
    """NaN, infinite and negative lengths, boundaries in no order (some bucket then, no fault)."""
    import batmobile
    r = torch.tensor([float("nan"), float("inf"), -float("inf"), -1.0, 5.0, 0.0])
    table = torch.randn(4, 3, generator=gen(1))
    bound = torch.tensor([1.0, 2.0, 3.0])
    out = batmobile.distance_bias(r.to(dev), bound.to(dev), table.to(dev), 5.0)
    assert torch.isnan(out[0]).all() and torch.isneginf(out[[1, 2, 4]]).all()
    assert torch.equal(out[5].cpu(), table[0])
    plain = batmobile.distance_bias(r.to(dev), bound.to(dev), table.to(dev))
    assert torch.isnan(plain[0]).all()
    assert torch.equal(plain[[1, 2, 3, 4, 5]].cpu(), table[[3, 0, 0, 3, 0]])
    mixed = batmobile.distance_bias(torch.rand(500, device=dev) * 4, bound[[2, 0, 1]].to(dev),
                                    table.to(dev))
    assert all(any(torch.equal(row, t) for t in table.to(dev)) for row in mixed[:20])


def test_distance_bias_strided_inputs(dev):
    import batmobile
    r, bound, table, g = _bias_inputs(600, 40, 8, 3)
    a = [t.to(dev).requires_grad_(True) for t in (r, table)]
    want = torch.autograd.grad(batmobile.distance_bias(a[0], bound.to(dev), a[1], 5.0), a, g.to(dev))
    wide = torch.stack([r, r], 1).to(dev)[:, 1].requires_grad_(True)
    turned = table.t().contiguous().to(dev).t().requires_grad_(True)
    out = batmobile.distance_bias(wide, torch.stack([bound, bound], 1).to(dev)[:, 0], turned, 5.0)
    got = torch.autograd.grad(out, [wide, turned], g.t().contiguous().to(dev).t())
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = torch.autograd.grad(batmobile.distance_bias(a[0], bound.to(dev), a[1], 5.0).sum(), a)
    full = torch.autograd.grad(batmobile.distance_bias(a[0], bound.to(dev), a[1], 5.0), a,
                               torch.ones(600, 8, device=dev))
    assert all(torch.equal(x, y) for x, y in zip(one, full))


@pytest.mark.parametrize("k", [-90, 90])
def test_distance_bias_scaled(dev, k):
    """All lengths times 2^k: the same bias, and the gradient times 2^-k, bit for bit."""
    import batmobile
    r, bound, table, g = [t.to(dev) for t in _bias_inputs(600, 40, 8, 3)]

    def run(scale):
        a = (r * scale).requires_grad_(True)
        out = batmobile.distance_bias(a, bound * scale, table, 5.0 * scale)
        return out, torch.autograd.grad(out, a, g)[0] * scale

    for got, want in zip(run(2.0 ** k), run(1.0)):
        assert torch.equal(got, want)


def test_distance_bias_single_gradients(dev):
    """Only the gradient that is wanted."""
    import batmobile
    r, bound, table, g = [t.to(dev) for t in _bias_inputs(300, 20, 4, 4)]
    both = [r.clone().requires_grad_(True), table.clone().requires_grad_(True)]
    want = torch.autograd.grad(batmobile.distance_bias(both[0], bound, both[1], 5.0), both, g)
    assert torch.equal(torch.autograd.grad(
        batmobile.distance_bias(both[0], bound, table, 5.0), both[0], g)[0], want[0])
    assert torch.equal(torch.autograd.grad(
        batmobile.distance_bias(r, bound, both[1], 5.0), both[1], g)[0], want[1])


def test_distance_bias_past_32_bits(dev):
    """More than 2^31 values."""
    import batmobile
    e, h = (1 << 25) + 77, 64
    r = torch.rand(e, generator=torch.Generator(device=dev).manual_seed(1), device=dev) * 5
    bound, table = torch.arange(1, 32, device=dev) * (5 / 32), torch.randn(32, h, device=dev)
    out = batmobile.distance_bias(r, bound, table)
    k = torch.bucketize(r[-1000:], bound, right=True)
    assert torch.equal(out[-1000:], table[k])
    t = table.requires_grad_(True)
    gt, = torch.autograd.grad(batmobile.distance_bias(r, bound, t), t, torch.ones_like(out))
    # counts of a million: a sum of ones is exact in fp32
    assert torch.equal(gt[:, 0].long(), torch.bincount(torch.bucketize(r, bound, right=True),
                                                       minlength=32))


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def _check_ln(dev, x, weight, bias, g, dtype, eps=1e-5):
    import batmobile
    leaf = [t.to(dev).requires_grad_(True) for t in (weight,) + ((bias,) if bias is not None else ())]
    xd = x.requires_grad_(True)
    out = batmobile.layer_norm(xd, leaf[0], leaf[1] if bias is not None else None, eps)
    grads = torch.autograd.grad(out, [xd] + leaf, g.to(dev))
    d = x.shape[-1]
    want, gx, gw, gb = ol.layer_norm(_np(x).reshape(-1, d), _np(weight), _np(bias), eps,
                                     _np(g).reshape(-1, d))
    r = 3e-6 + (ROUND[dtype] if dtype == "bf16" else 0)
    assert out.dtype == x.dtype and out.shape == x.shape and grads[0].shape == x.shape
    assert normwise_err(_np(out).reshape(-1, d), want) <= r
    # gx = rs (u - mean u - xh mean(u xh)): the three terms cancel for few elements (for two
    # nearly wholly), so the error is measured by the terms.  |mean u| <= max |u|, and |mean(u xh)| <= max |u|
    # as xh has mean square 1 at most
    x2, u = _np(x).reshape(-1, d), np.abs(_np(g).reshape(-1, d) * _np(weight))
    dev2 = x2 - x2.mean(1, keepdims=True)
    rs = 1 / np.sqrt((dev2 ** 2).mean(1, keepdims=True) + eps)
    terms = rs * (u + u.max(1, keepdims=True) * (1 + np.abs(dev2) * rs))
    _within(grads[0].reshape(-1, d), gx, 3e-6 * terms + (r - 3e-6) * np.abs(gx))
    # sums over the rows, xh to 3e-6 of its largest (at most the root of d)
    rows = want.shape[0]
    absum = np.abs(_np(g).reshape(-1, d)).sum(0)
    _within(grads[1], gw, absum * (3e-6 * min(d, 64) ** 0.5 + (rows + 8) * U * d ** 0.5) + 1e-30)
    if bias is not None:
        _within(grads[2], gb, absum * (rows + 8) * U + 1e-30)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (5, 3), (33, 7), (64, 8), (9, 9), (130, 16),
                                    (7, 31), (65, 32), (66, 33), (1000, 64), (37, 100), (17, 127),
                                    (40, 128), (5, 129), (20, 256), (6, 257), (9, 500), (8, 512),
                                    (5, 1000), (4, 1024), (3, 1025), (5, 2048), (3, 2049), (3, 4096),
                                    (2, 4100), (2, 4099), (3, 8192), (2, 8191)])
def test_layer_norm(dev, dtype, rows, d):
    g = gen(rows + d)
    x = (torch.randn(rows, d, generator=g) + 0.5).to(TYPES[dtype]).to(dev)
    _check_ln(dev, x, torch.randn(d, generator=g), torch.randn(d, generator=g),
              torch.randn(rows, d, generator=g).to(TYPES[dtype]), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,d", [(1, 8), (3, 33), (5, 100), (33, 64), (7, 500), (2, 2048)])
def test_layer_norm_without_eps(dev, dtype, rows, d):
    """eps = 0: a workgroup's places without a row have no part in the weights' gradient."""
    g = gen(rows + d)
    x = (torch.randn(rows, d, generator=g) + 0.5).to(TYPES[dtype]).to(dev)
    _check_ln(dev, x, torch.randn(d, generator=g), torch.randn(d, generator=g),
              torch.randn(rows, d, generator=g).to(TYPES[dtype]), dtype, eps=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form", ["scalars", "columns", "rows", "offset", "three", "expanded", "packed"])
def test_layer_norm_strides(dev, dtype, form):
    g = gen(11)
    t = TYPES[dtype]
    if form == "scalars":
        x = torch.randn(21, 40, 16, generator=g).to(t).to(dev)[:, :, 0]
    elif form == "columns":
        x = torch.randn(40, 21, generator=g).to(t).to(dev).t()
    elif form == "rows":
        x = torch.randn(42, 48, generator=g).to(t).to(dev)[::2, :40]
    elif form == "offset":
        x = torch.randn(21 * 40 + 3, generator=g).to(t).to(dev)[3:].view(21, 40)
    elif form == "three":
        x = torch.randn(5, 7, 40, generator=g).to(t).to(dev)
    elif form == "expanded":
        x = torch.randn(1, 40, generator=g).to(t).to(dev).expand(21, 40)
    else:
        x = torch.randn(7, 5, 40, generator=g).to(t).to(dev).transpose(0, 1)
    x = x.detach()
    _check_ln(dev, x, torch.randn(40, generator=g), torch.randn(40, generator=g),
              torch.randn(x.shape, generator=g).to(t), dtype)


def test_layer_norm_far_from_zero(dev):
    """Rows whose mean is 10,000 times their spread keep their digits: the inputs' own are the limit."""
    g = gen(12)
    x = (torch.randn(50, 96, generator=g) + 1e4).to(dev)
    _check_ln(dev, x, torch.randn(96, generator=g), None, torch.randn(50, 96, generator=g), "f32")


def test_layer_norm_constant_rows(dev):
    import batmobile
    w, b = torch.randn(24, generator=gen(13)).to(dev), torch.randn(24, generator=gen(14)).to(dev)
    x = torch.full((3, 24), 7.0, device=dev)
    # what is left of 7 - mean: 2^-24 of its own rounding, times 1 / sqrt(eps) = 316
    assert (batmobile.layer_norm(x, w, b) - b).abs().max() <= 2.0 ** -22 * float(b.abs().max())
    assert batmobile.layer_norm(x, w).abs().max() <= 7 * 2.0 ** -46 * 316 * float(w.abs().max())


def test_layer_norm_empty_and_large(dev):
    import batmobile
    w = torch.randn(32, device=dev, requires_grad=True)
    x = torch.zeros(0, 32, device=dev, requires_grad=True)
    gx, gw = torch.autograd.grad(batmobile.layer_norm(x, w).sum(), [x, w])
    assert gx.shape == (0, 32) and torch.equal(gw, torch.zeros(32, device=dev))
    rows, d = (1 << 20) + 5, 2048                      # more than 2^31 elements
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=dev).fill_(1.0)
    x[-3:] = torch.randn(3, d, generator=gen(15)).bfloat16().to(dev)
    w = torch.ones(d, device=dev)
    y = batmobile.layer_norm(x, w)
    want = ol.layer_norm(_np(x[-3:]), _np(w))
    assert normwise_err(_np(y[-3:]), want) <= 3e-6 + 2.0 ** -8
    assert not y[:-3:100003].any()
    gx, gw, gb = _batmobile.layer_norm_backward(y, x, w, True, 1e-5)
    want = ol.layer_norm(_np(x[-3:]), _np(w), None, 1e-5, _np(y[-3:]))
    assert normwise_err(_np(gx[-3:]), want[1]) <= 3e-6 + 2.0 ** -8 * 4
    assert normwise_err(_np(gw), want[2]) <= 1e-5 and normwise_err(_np(gb), want[3]) <= 1e-5


# ---------------------------------------------------------------------------
# channel mixing
# ---------------------------------------------------------------------------

def _features(n, c, dtype, seed):
    g = gen(seed)
    scale = torch.tensor([1.0] + [0.7] * 3 + [0.5] * 5 + [0.3] * 7)
    return (torch.randn(n, c, 16, generator=g) * scale
            * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g))).to(TYPES[dtype])


def _check_mixing(dev, n, c, o, dtype, kept, seed):
    import batmobile
    x, gy = _features(n, c, dtype, seed), _features(n, o, dtype, seed + 1)
    w = torch.randn(4, c, o, generator=gen(seed + 2)) / c ** 0.5
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = batmobile.channel_mixing(xd, wd, kept)
    gx, gw = torch.autograd.grad(y, [xd, wd], gy.to(dev))
    kx = ol.kept(_np(x)) if kept else _np(x)
    want, wx, ww = ol.channel_mixing(_np(x), _np(w), _np(gy), kx)
    ay, ax, aw = ol.channel_mixing(np.abs(_np(x)), np.abs(_np(w)), np.abs(_np(gy)), np.abs(kx))
    more = 2.0 ** -15 if dtype == "bf16" else 0.0
    out = ROUND[dtype] if dtype == "bf16" else 0.0
    _within(y, want, ay * ((c + 16) * U + more) + np.abs(want) * out)
    _within(gx, wx, ax * ((o + 16) * U + more) + np.abs(wx) * out)
    terms = n * np.array([1, 3, 5, 7])[:, None, None]
    _within(gw, ww, aw * (terms + 16) * U)
    # as a whole the rounding errors do not add up one way
    assert normwise_err(_np(gw), ww) <= 3e-6
    assert normwise_err(_np(y), want) <= 3e-6 + out and normwise_err(_np(gx), wx) <= 3e-6 + out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kept", [None, "e4m3"])
@pytest.mark.parametrize("n,c,o", [(1, 1, 1), (2, 3, 5), (15, 16, 16), (16, 31, 33), (17, 32, 32),
                                   (33, 64, 64), (100, 40, 100), (31, 100, 200), (65, 128, 64),
                                   (32, 130, 129), (40, 256, 8), (200, 8, 256), (129, 33, 65),
                                   (21, 300, 70), (50, 70, 300)])
def test_channel_mixing(dev, dtype, kept, n, c, o):
    _check_mixing(dev, n, c, o, dtype, kept, n + c + o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_channel_mixing_widest(dev, dtype):
    _check_mixing(dev, 3, 2048, 17, dtype, "e4m3", 1)
    _check_mixing(dev, 3, 17, 2048, dtype, None, 2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_channel_mixing_many_atoms(dev, dtype):
    """More ranges of atoms than one in the weight's gradient, and an odd end."""
    _check_mixing(dev, 3001, 24, 40, dtype, None, 3)
    _check_mixing(dev, 3001, 24, 40, dtype, "e4m3", 4)


def test_channel_mixing_empty(dev):
    import batmobile
    for kept in (None, "e4m3"):
        x = torch.zeros(0, 8, 16, device=dev, requires_grad=True)
        w = torch.randn(4, 8, 5, device=dev, requires_grad=True)
        y = batmobile.channel_mixing(x, w, kept)
        gx, gw = torch.autograd.grad(y.sum(), [x, w])
        assert y.shape == (0, 5, 16) and gx.shape == x.shape
        assert torch.equal(gw, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_channel_mixing_strides(dev, dtype):
    """Slices, transposes and odd addresses give what their copies give, bit for bit."""
    import batmobile
    x = _features(20, 30, dtype, 5).to(dev)
    w = torch.randn(4, 30, 12, generator=gen(6)).to(dev)
    gy = _features(20, 12, dtype, 7).to(dev)

    def run(x, w, gy):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = batmobile.channel_mixing(x, w, "e4m3")
        return (y.detach(),) + torch.autograd.grad(y, [x, w], gy)

    want = run(x, w, gy)
    flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=dev)
    flat[1:] = x.flatten()
    forms = [x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x], 1)[:, 30:],
             flat[1:].view_as(x)]
    for v in forms:
        got = run(v, w.transpose(1, 2).contiguous().transpose(1, 2),
                  gy.transpose(1, 2).contiguous().transpose(1, 2))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("c", [33, 70, 300])
def test_channel_mixing_infinities(dev, c):
    """An infinity or NaN reaches what it is a term of, and nothing else."""
    import batmobile
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(40, c, 16, generator=gen(8)).to(dev, dtype)
        w = (torch.rand(4, c, 20, generator=gen(9)) + 0.5).to(dev)
        want = batmobile.channel_mixing(x, w)
        x[5, 7, 3], x[33, c - 1, 9] = float("inf"), float("nan")
        y = batmobile.channel_mixing(x, w)
        assert torch.isinf(y[5, :, 3]).all() and torch.isnan(y[33, :, 9]).all()
        y[5, :, 3], y[33, :, 9] = want[5, :, 3], want[33, :, 9]
        assert torch.equal(y, want)
        x = torch.rand(40, c, 16, generator=gen(8)).to(dev, dtype) + 0.5
        want = batmobile.channel_mixing(x, w)
        w[1, 6, 4] = -float("inf")
        y = batmobile.channel_mixing(x, w)
        assert torch.isneginf(y[:, 4, 1:4]).all()
        y[:, 4, 1:4] = want[:, 4, 1:4]
        assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("c", [20, 64, 70, 128, 200, 256, 300])
def test_channel_mixing_infinities_times_round_weights(dev, dtype, c):
    """Weights of which nothing is left behind their leading bits, zeros among them: an infinity times
    zero is no number, any other weight gives its sign's infinity."""
    import batmobile
    x = torch.randint(-4, 5, (35, c, 16), generator=gen(41)).to(TYPES[dtype])
    w = torch.tensor([1.0, -2.0, 0.5, -(2.0 ** -100), 1.5, 0.0, -0.0, 2.0 ** 100])
    w = w[torch.randint(0, 8, (4, c, 24), generator=gen(42))]
    w[:, 1, :8] = torch.tensor([1.0, -2.0, 0.5, -(2.0 ** -100), 1.5, 0.0, -0.0, 2.0 ** 100])
    x[3, 1, 0], x[20, 1, 5], x[34, 1, 15] = float("inf"), -float("inf"), float("inf")
    y = _np(batmobile.channel_mixing(x.to(dev), w.to(dev)))
    with np.errstate(invalid="ignore"):
        for n, m, l in ((3, 0, 0), (20, 5, 2), (34, 15, 3)):
            want = np.float64(x[n, 1, m]) * w[l, 1].double().numpy()
            assert np.array_equal(y[n, :, m], want, equal_nan=True)
    assert np.isfinite(np.delete(y, [3, 20, 34], 0)).all()
    back = _np(_batmobile.channel_mixing(x.to(dev), w.transpose(1, 2).contiguous().to(dev), True))
    assert np.array_equal(back, y, equal_nan=True)


@pytest.mark.parametrize("kept", [None, "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_weight_gradient_with_nan(dev, dtype, kept):
    """A NaN in x or in the gradient reaches its channel's row or column of its degree alone."""
    import batmobile
    x, g = _features(37, 20, dtype, 12).to(dev), _features(37, 70, dtype, 13).to(dev)
    w = torch.randn(4, 20, 70, generator=gen(14)).to(dev).requires_grad_(True)
    want, = torch.autograd.grad(batmobile.channel_mixing(x, w, kept), w, g)
    x[36, 19, 5], g[20, 69, 12] = float("nan"), float("nan")
    got, = torch.autograd.grad(batmobile.channel_mixing(x, w, kept), w, g)
    bad = torch.isnan(got)
    hit = torch.zeros_like(bad)
    hit[2, 19], hit[3, :, 69] = True, True
    assert torch.equal(bad, hit)
    # the 8-bit block that holds the NaN is another one: its largest value may have gone
    hit[:, 16:] = hit[:, 16:] | (kept is not None)
    assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_channel_mixing_single_gradients(dev, dtype):
    """Only the gradient that is wanted, the same as with both; nothing is kept for the other."""
    import batmobile
    x, g = _features(33, 24, dtype, 15).to(dev), _features(33, 10, dtype, 16).to(dev)
    w = torch.randn(4, 24, 10, generator=gen(17)).to(dev)
    both = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    want = torch.autograd.grad(batmobile.channel_mixing(*both), both, g)
    y = batmobile.channel_mixing(both[0], w)
    z = batmobile.channel_mixing(x, both[1])
    w.mul_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, both[0], g)
    assert torch.equal(torch.autograd.grad(z, both[1], g)[0], want[1])
    y = batmobile.channel_mixing(both[0], w)
    both[0].detach().zero_()                           # its values are not needed
    assert torch.equal(torch.autograd.grad(y, both[0], g)[0], want[0])


def test_buckets_of_the_backward_stay_in_bounds(dev):
    """Buckets that no forward gave are taken to the last one, or left out; nothing is written past."""
    k = torch.tensor([0, 1, 5, 300, -1], dtype=torch.int16, device=dev)
    g = torch.ones(5, 2, device=dev)
    for buckets in (2, 200):
        gt, gl = _batmobile.distance_bias_backward(None, k, g, buckets, 0.0, True, False)
        assert gl is None and gt.shape == (buckets, 2) and torch.isfinite(gt).all()
        assert gt[0, 0] >= 1 and gt.sum() <= 10


def test_channel_mixing_past_32_bits(dev):
    """More than 2^31 elements, and a launch of more than 2^24 atoms."""
    import batmobile
    n = (1 << 24) + 37
    x = torch.ones(n, 9, 16, dtype=torch.bfloat16, device=dev)
    x[-40:] = _features(40, 9, "bf16", 10).to(dev)
    w = torch.randn(4, 9, 3, generator=gen(11))
    y = batmobile.channel_mixing(x, w.to(dev))
    want = ol.channel_mixing(_np(x[-40:]), _np(w))
    assert normwise_err(_np(y[-40:]), want) <= 2.0 ** -8 + 1e-5
    assert torch.equal(y[1], y[n - 50])
    gw = _batmobile.channel_mixing_weight_grad(x, None, None, y)
    total = _np(y[:-40, 0, 0].double().sum()) + (_np(x[-40:, 4, 0]) * _np(y[-40:, 0, 0])).sum()
    assert abs(float(gw[0, 4, 0]) - total) <= 1e-5 * abs(total)


# ---------------------------------------------------------------------------
# 8 bits
# ---------------------------------------------------------------------------

def _awkward(n, c, dtype, seed):
    """Ties, subnormal codes, zeros, not finite, largest and least values."""
    g = gen(seed)
    x = torch.randn(n, c, 16, generator=g) * 10.0 ** torch.randint(-38, 38, (n, c, 1), generator=g)
    x[0] = torch.round(x[0].sign() * torch.rand(c, 16, generator=g) * 64) / 16
    x[0, 0, 0] = 448.0
    x[1] = 0.0
    x[1, 0, 5] = -0.0
    x[2, 0, 0], x[2, 0, 1], x[2, 0, 2] = float("inf"), -float("inf"), float("nan")
    x[3, 0, 0], x[3, 0, 1] = 3.4e38, 1e-40
    x[4] *= 1e-38
    return x.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c", [(5, 1), (6, 7), (40, 8), (9, 20), (33, 64), (5, 2048)])
def test_checkpoint(dev, dtype, n, c):
    """Codes and exponents bit for bit, and what they hold."""
    import batmobile
    x = _awkward(n, c, dtype, n + c)
    codes, exps = batmobile.checkpoint_encode(x.to(dev))
    wc, we = ol.encode(_np(x))
    assert codes.dtype == torch.float8_e4m3fn and torch.equal(exps.cpu(), torch.from_numpy(we))
    got = codes.view(torch.uint8).cpu().numpy()
    nan = (wc & 127) == 127
    assert np.array_equal((got & 127) == 127, nan) and np.array_equal(got[~nan], wc[~nan])
    for t in (torch.float32, torch.bfloat16):
        back = batmobile.checkpoint_decode(codes, exps, t)
        want = ol.decode(wc, we)
        assert back.dtype == t
        assert np.array_equal(_np(back), want, equal_nan=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_checkpoint_largest(dev, dtype):
    """Where codes end: the halves between 240, 256 and 448 times 2^120, and the largest numbers."""
    import batmobile
    big = torch.finfo(TYPES[dtype]).max
    x = torch.zeros(2, 8, 16)
    x[0, 0, :6] = torch.tensor([248.0, -248.0, 232.0, 224.0, 249.0, 1.0]) * 2.0 ** 120
    x[1, 3, :4] = torch.tensor([big, -big, 240 * 2.0 ** 120, 216 * 2.0 ** 120])
    x = x.to(TYPES[dtype])
    codes, exps = batmobile.checkpoint_encode(x.to(dev))
    wc, we = ol.encode(_np(x))
    assert torch.equal(exps.cpu(), torch.from_numpy(we))
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), wc)
    back = batmobile.checkpoint_decode(codes, exps)
    assert torch.isfinite(back).all()
    assert (np.abs(_np(back) - _np(x)) <= 2.0 ** -4 * np.abs(_np(x))).all()


def test_checkpoint_empty(dev):
    import batmobile
    codes, exps = batmobile.checkpoint_encode(torch.zeros(0, 9, 16, device=dev))
    assert codes.shape == (0, 9, 16) and exps.shape == (0, 2)
    assert batmobile.checkpoint_decode(codes, exps).shape == (0, 9, 16)


# ---------------------------------------------------------------------------
# gated activation
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kept", [None, "e4m3"])
@pytest.mark.parametrize("n,c", [(1, 1), (3, 5), (17, 8), (40, 20), (129, 64), (7, 100), (3, 2048)])
def test_gate_activation(dev, dtype, kept, n, c):
    import batmobile
    x, g = 3 * _features(n, c, dtype, n + c).float(), _features(n, c, dtype, n + c + 1)
    if n > 2:
        x[0, 0, 0], x[1, 0, 0], x[2, 0, 0] = 30.0, -30.0, -100.0
    x = x.to(TYPES[dtype])
    xd = x.to(dev).requires_grad_(True)
    y = batmobile.gate_activation(xd, kept)
    gx, = torch.autograd.grad(y, xd, g.to(dev))
    kx = ol.kept(_np(x)) if kept else _np(x)
    want, wx = ol.gate_activation(_np(x), _np(g), kx)
    out = ROUND[dtype] if dtype == "bf16" else 0.0
    _within(y, want, np.abs(want) * (16 * U + out) + 1e-37)
    on = 1 / (1 + np.exp(-kx[:, :, :1]))
    terms = on * np.abs(_np(g))
    terms[:, :, :1] += on / (1 + np.exp(kx[:, :, :1])) * np.abs(_np(g) * kx).sum(2, keepdims=True)
    _within(gx, wx, terms * 24 * U + np.abs(wx) * out + 1e-37)


def test_gate_activation_empty_and_strided(dev):
    import batmobile
    x = torch.zeros(0, 4, 16, device=dev, requires_grad=True)
    gx, = torch.autograd.grad(batmobile.gate_activation(x, "e4m3").sum(), x)
    assert gx.shape == x.shape
    x = _features(12, 20, "bf16", 3).to(dev)
    for v in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x], 1)[:, 20:]):
        assert torch.equal(batmobile.gate_activation(v), batmobile.gate_activation(x))


def test_gate_activation_past_32_bits(dev):
    import batmobile
    n, c = (1 << 20) + 3, 136                          # 2^31 elements and some
    x = torch.ones(n, c, 16, dtype=torch.bfloat16, device=dev)
    x[-2:] = _features(2, c, "bf16", 4).to(dev)
    y = batmobile.gate_activation(x)
    want = ol.gate_activation(_np(x[-2:]))
    assert normwise_err(_np(y[-2:]), want) <= 2.0 ** -8 + 1e-6
    codes, exps = batmobile.checkpoint_encode(x)
    assert np.array_equal(_np(batmobile.checkpoint_decode(codes[-2:], exps[-2:])), ol.kept(_np(x[-2:])))


# ---------------------------------------------------------------------------
# all of them
# ---------------------------------------------------------------------------

def _calls(dev, seed=21):
    """{name: (call of the leaves, leaves)} of each operator with gradients, small."""
    import batmobile
    g = gen(seed)
    r = (5 * torch.rand(300, generator=g)).to(dev)
    bound = torch.linspace(0.5, 4.5, 9).to(dev)
    t = lambda *s: torch.randn(*s, generator=g).to(dev)          # noqa: E731
    return {
        "distance_bias": (lambda r, tab: batmobile.distance_bias(r, bound, tab, 6.0), [r, t(10, 4)]),
        "layer_norm": (batmobile.layer_norm, [t(50, 24), t(24), t(24)]),
        "channel_mixing": (batmobile.channel_mixing, [t(40, 12, 16), t(4, 12, 20)]),
        "channel_mixing_e4m3": (lambda x, w: batmobile.channel_mixing(x, w, "e4m3"),
                                [t(40, 12, 16), t(4, 12, 20)]),
        "gate_activation": (batmobile.gate_activation, [t(40, 12, 16)]),
        "gate_activation_e4m3": (lambda x: batmobile.gate_activation(x, "e4m3"), [t(40, 12, 16)]),
    }


NAMES = ["distance_bias", "layer_norm", "channel_mixing", "channel_mixing_e4m3", "gate_activation",
         "gate_activation_e4m3"]


def _step(call, leaves):
    out = call(*leaves)
    return (out.detach(),) + torch.autograd.grad(out, leaves, torch.ones_like(out))


@pytest.mark.parametrize("name", NAMES)
def test_same_from_run_to_run_and_on_another_stream(dev, name):
    call, leaves = _calls(dev)[name]
    leaves = [t.requires_grad_(True) for t in leaves]
    want = _step(call, leaves)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        with torch.cuda.stream(stream):
            got = _step(call, leaves)
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_captured_step(dev, name):
    """Forward and backward in a graph, replayed with other inputs between eager work."""
    call, leaves = _calls(dev)[name]
    leaves = [t.requires_grad_(True) for t in leaves]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(call, leaves)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(call, leaves)
    for k in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9).add_(0.01 * k)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(call, leaves)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k


@pytest.mark.parametrize("name", NAMES)
def test_two_calls_before_either_backward(dev, name):
    """What a call keeps is its own."""
    call, leaves = _calls(dev)[name]
    other = [t.clone().mul_(0.5).requires_grad_(True) for t in leaves]
    leaves = [t.requires_grad_(True) for t in leaves]
    want = _step(call, leaves), _step(call, other)
    a, b = call(*leaves), call(*other)
    gb = torch.autograd.grad(b, other, torch.ones_like(b))
    ga = torch.autograd.grad(a, leaves, torch.ones_like(a))
    assert all(torch.equal(x, y) for x, y in zip(ga, want[0][1:]))
    assert all(torch.equal(x, y) for x, y in zip(gb, want[1][1:]))


@pytest.mark.parametrize("name", NAMES)
def test_no_second_derivatives(dev, name):
    call, leaves = _calls(dev)[name]
    leaves = [t.requires_grad_(True) for t in leaves]
    grads = torch.autograd.grad(call(*leaves).square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        sum(t.sum() for t in grads).backward()


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(dev, name):
    call, leaves = _calls(dev)[name]
    with torch.inference_mode():
        got = call(*leaves)
    assert torch.equal(got, call(*leaves))


def test_an_input_changed_before_the_backward(dev):
    """In 8 bits the layer has its own copy; as it is, autograd refuses."""
    import batmobile
    x = torch.randn(20, 8, 16, generator=gen(31)).to(dev)
    w = torch.randn(4, 8, 8, generator=gen(32)).to(dev).requires_grad_(True)
    g = torch.randn(20, 8, 16, generator=gen(33)).to(dev)
    want, = torch.autograd.grad(batmobile.channel_mixing(x, w, "e4m3"), w, g)
    y, z = batmobile.channel_mixing(x, w, "e4m3"), batmobile.channel_mixing(x, w)
    x.zero_()
    assert torch.equal(torch.autograd.grad(y, w, g)[0], want)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(z, w, g)


def test_memory_of_checkpoints(dev):
    """What a layer holds for the backward: 1 + 1/128 bytes a value, and the result."""
    import batmobile
    x = torch.randn(4096, 64, 16, device=dev)
    w = torch.randn(4, 64, 64, device=dev, requires_grad=True)
    for call in (lambda: batmobile.gate_activation(x.detach().requires_grad_(True), "e4m3"),
                 lambda: batmobile.channel_mixing(x, w, "e4m3")):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = call()
        held = torch.cuda.memory_allocated() - before - y.numel() * 4
        assert held <= x.numel() * (1 + 1 / 128) + 4096
        del y


def test_refusals(dev):
    import batmobile as bm
    f = lambda *s, **k: torch.zeros(*s, device=dev, **k)           # noqa: E731
    bad = [
        ("lengths", lambda: bm.distance_bias(f(3, 1), f(2), f(3, 4))),
        ("float32", lambda: bm.distance_bias(f(3, dtype=torch.float64), f(2), f(3, 4))),
        ("boundaries", lambda: bm.distance_bias(f(3), f(3), f(3, 4))),
        ("table", lambda: bm.distance_bias(f(3), f(2), f(12))),
        ("table", lambda: bm.distance_bias(f(3), f(4096), f(4097, 1))),
        ("table", lambda: bm.distance_bias(f(3), f(2), f(3, 1025))),
        ("cutoff", lambda: bm.distance_bias(f(3), f(2), f(3, 4), 0.0)),
        ("cutoff", lambda: bm.distance_bias(f(3), f(2), f(3, 4), -1.0)),
        ("cutoff", lambda: bm.distance_bias(f(3), f(2), f(3, 4), float("nan"))),
        ("cutoff", lambda: bm.distance_bias(f(3), f(2), f(3, 4), 1e300)),
        ("boundaries", lambda: bm.distance_bias(f(3), f(2, requires_grad=True), f(3, 4))),
        ("must be on", lambda: bm.distance_bias(f(3), torch.zeros(2), f(3, 4))),
        ("x must be", lambda: bm.layer_norm(f(3, 0), f(0))),
        ("x must be", lambda: bm.layer_norm(f(3, 8193), f(8193))),
        ("x must be", lambda: bm.layer_norm(f(()), f(1))),
        ("weight", lambda: bm.layer_norm(f(3, 4), f(5))),
        ("float32", lambda: bm.layer_norm(f(3, 4), f(4, dtype=torch.bfloat16))),
        ("bias", lambda: bm.layer_norm(f(3, 4), f(4), f(1, 4))),
        ("eps", lambda: bm.layer_norm(f(3, 4), f(4), eps=-1.0)),
        ("float32 or bfloat16", lambda: bm.layer_norm(f(3, 4, dtype=torch.float16), f(4))),
        ("3D", lambda: bm.channel_mixing(f(3, 8, 9), f(4, 8, 8))),
        ("weight", lambda: bm.channel_mixing(f(3, 8, 16), f(4, 9, 8))),
        ("weight", lambda: bm.channel_mixing(f(3, 8, 16), f(3, 8, 8))),
        ("channels", lambda: bm.channel_mixing(f(3, 8, 16), f(4, 8, 2049))),
        ("channels", lambda: bm.channel_mixing(f(1, 2049, 16), f(4, 2049, 8))),
        ("channels", lambda: bm.channel_mixing(f(3, 0, 16), f(4, 0, 8))),
        ("float32", lambda: bm.channel_mixing(f(3, 8, 16), f(4, 8, 8, dtype=torch.bfloat16))),
        ("checkpoint", lambda: bm.channel_mixing(f(3, 8, 16), f(4, 8, 8), "e5m2")),
        ("checkpoint", lambda: bm.gate_activation(f(3, 8, 16), "int8")),
        ("3D", lambda: bm.gate_activation(f(3, 8))),
        ("float32 or bfloat16", lambda: bm.gate_activation(f(3, 8, 16, dtype=torch.float16))),
        ("codes", lambda: bm.checkpoint_decode(f(3, 8, 16), f(3, 1, dtype=torch.uint8))),
        ("exponents", lambda: bm.checkpoint_decode(f(3, 8, 16).to(torch.float8_e4m3fn), f(3, 1))),
        ("exponents", lambda: bm.checkpoint_decode(f(3, 9, 16).to(torch.float8_e4m3fn),
                                                   f(3, 1, dtype=torch.uint8))),
        ("dtype", lambda: bm.checkpoint_decode(f(3, 8, 16).to(torch.float8_e4m3fn),
                                               f(3, 1, dtype=torch.uint8), torch.float16)),
    ]
    for match, call in bad:
        with pytest.raises(RuntimeError, match=match):
            call()
