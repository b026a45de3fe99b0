"""The oracle of the operators beside attention: by definition, and its gradients against differences."""
import numpy as np
import pytest

from oracle import block as ob
from oracle import layers as ol


def _difference(f, x, g, h=1e-6):
    """sum g df/dx by central differences."""
    out = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        out[i] = ((f(a) - f(b)) * g).sum() / (2 * h)
    return out


def _rng(seed):
    return np.random.default_rng(seed)


@pytest.mark.parametrize("cutoff", [None, 2.0])
def test_distance_bias(cutoff):
    rng = _rng(1)
    r = rng.uniform(0.05, 1.9, 20)
    bound, table = np.linspace(0.3, 1.8, 6), rng.normal(size=(7, 3))
    g = rng.normal(size=(20, 3))
    out, gt, gr = ol.distance_bias(r, bound, table, cutoff, g)
    for e in range(20):
        want = table[sum(b <= r[e] for b in bound)]
        if cutoff:
            want = want + np.log(1 - (r[e] / cutoff) ** 2)
        assert np.allclose(out[e], want, rtol=0, atol=1e-13)
    assert np.allclose(gt, _difference(lambda t: ol.distance_bias(r, bound, t, cutoff), table, g),
                       atol=1e-7)
    assert np.allclose(gr, _difference(lambda t: ol.distance_bias(t, bound, table, cutoff), r, g),
                       atol=1e-6)


def test_distance_bias_edges():
    """A boundary belongs to the bucket above it; from the cutoff on -inf, and no gradient."""
    out, _, gr = ol.distance_bias([1.0, 0.999, 2.0, 3.0, np.nan], [1.0], [[5.0], [7.0]], 2.0,
                                  np.ones((5, 1)))
    assert out[0, 0] == 7 + np.log(0.75) and out[1, 0] < 5
    assert np.isneginf(out[2, 0]) and np.isneginf(out[3, 0]) and np.isnan(out[4, 0])
    assert gr[2] == 0 and gr[3] == 0 and gr[0] < 0


def test_layer_norm():
    rng = _rng(2)
    x, w, b = rng.normal(size=(4, 7)), rng.normal(size=7), rng.normal(size=7)
    g = rng.normal(size=(4, 7))
    y, gx, gw, gb = ol.layer_norm(x, w, b, 1e-5, g)
    for i in range(4):
        assert np.allclose(y[i], (x[i] - x[i].mean()) / np.sqrt(x[i].var() + 1e-5) * w + b)
    assert np.allclose(gx, _difference(lambda t: ol.layer_norm(t, w, b), x, g), atol=1e-7)
    assert np.allclose(gw, _difference(lambda t: ol.layer_norm(x, t, b), w, g), atol=1e-7)
    assert np.allclose(gb, _difference(lambda t: ol.layer_norm(x, w, t), b, g), atol=1e-7)


def test_channel_mixing():
    rng = _rng(3)
    x, w, g = rng.normal(size=(2, 3, 16)), rng.normal(size=(4, 3, 2)), rng.normal(size=(2, 2, 16))
    y, gx, gw = ol.channel_mixing(x, w, g)
    for m, l in enumerate(ob.DEGREE):
        assert np.allclose(y[:, :, m], x[:, :, m] @ w[l])
    assert np.allclose(gx, _difference(lambda t: ol.channel_mixing(t, w), x, g), atol=1e-7)
    assert np.allclose(gw, _difference(lambda t: ol.channel_mixing(x, t), w, g), atol=1e-7)
    z = rng.normal(size=x.shape)
    assert np.allclose(ol.channel_mixing(x, w, g, z)[2], ol.channel_mixing(z, w, g)[2])


def test_gate_activation():
    rng = _rng(4)
    x, g = rng.normal(size=(2, 3, 16)), rng.normal(size=(2, 3, 16))
    y, gx = ol.gate_activation(x, g)
    assert np.allclose(y, x / (1 + np.exp(-x[:, :, :1])))
    assert np.allclose(gx, _difference(ol.gate_activation, x, g), atol=1e-7)
    z = rng.normal(size=x.shape)
    assert np.allclose(ol.gate_activation(x, g, z)[1], ol.gate_activation(z, g)[1])


def test_e4m3_against_torch():
    import torch
    values = ol.e4m3_values()
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert np.array_equal(codes.float().numpy(), values)
    x = torch.randn(3, 16, 16, generator=torch.Generator().manual_seed(5))
    x[0, 0, 0], x[0, 1, 3] = 448.0, 1 + 1 / 16          # a block of power 2^0, a tie to even
    c, e = ol.encode(x.numpy())
    want = (x[0, :8] * 1.0).to(torch.float8_e4m3fn)
    assert e[0, 0] == 127 and np.array_equal(c[0, :8], want.view(torch.uint8).numpy())


def test_encode():
    rng = _rng(6)
    x = rng.normal(size=(5, 11, 16)) * 10.0 ** rng.integers(-30, 30, (5, 11, 1))
    c, e = ol.encode(x)
    v = ol.decode(c, e)
    top = np.stack([np.abs(x[:, 8 * b:8 * b + 8]).max((1, 2)) for b in range(2)], 1)
    scale = 2.0 ** (e.astype(float) - 127)
    assert (top <= 448 * scale).all() and (top > 224 * scale).all()
    s = np.repeat(scale, 8, 1)[:, :11, None]
    assert (np.abs(v - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s)).all()
    # not finite: NaN, and no part in the maximum; nothing but zeros: the least power
    x = np.zeros((1, 9, 16))
    x[0, 0, 0], x[0, 1, 1], x[0, 2, 2] = np.inf, np.nan, 3.0
    c, e = ol.encode(x)
    assert e[0, 0] == 127 - 7 and e[0, 1] == 127 - 110
    v = ol.decode(c, e)
    assert np.isnan(v[0, 0, 0]) and np.isnan(v[0, 1, 1]) and v[0, 2, 2] == 3.0


@pytest.mark.parametrize("top", [225.0, 300.0, 448.0])
def test_how_far_codes_are_off(top):
    """A value of 2^-6 2^E or more by 2^-4 of itself at most, a smaller one by 2^-10 2^E; in a block whose
    largest is just above 224 2^E, 2^-4 holds down to 2^-13.8 of it and no further."""
    rng = _rng(7)
    for k in (-100, 0, 100):
        x = np.exp2(rng.uniform(-16, 0, (40, 8, 16))) * rng.choice([-1, 1], (40, 8, 16)) * top * 2.0 ** k
        x[:, 0, 0] = top * 2.0 ** k
        c, e = ol.encode(x)
        assert (e == k + 127).all()
        off, unit = np.abs(ol.decode(c, e) - x), 2.0 ** k
        large = np.abs(x) >= 2.0 ** -6 * unit
        assert (off <= 2.0 ** -4 * np.abs(x))[large].all() and (off <= 2.0 ** -10 * unit)[~large].all()
        assert large[np.abs(x) >= 2.0 ** -13.8 * top * unit].all()
        small = ~large & (np.abs(x) >= 2.0 ** -15 * top * unit)
        assert (off > 2.0 ** -4 * np.abs(x))[small].any()
