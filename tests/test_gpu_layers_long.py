"""The operators beside attention where a workgroup goes on to further work: tiles of atoms, steps of a
range, batches of edges, launches after the first.  Every row differs from every other.

Bounds, u = 2^-24:
  mixing    a sum of K products, each as exact as one of fp32: (K + 16) u sum |x w|; bf16: the weight to
            2^-15, the result to 2^-8 of itself more
"""
import pytest
import torch

import _batmobile

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24
DEGREE = [0] + [1] * 3 + [2] * 5 + [3] * 7


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _features(dev, n, c, dtype, seed):
    g = _gen(dev, seed)
    return (torch.randn(n, c, 16, generator=g, device=dev)
            * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g, device=dev))).to(TYPES[dtype])


def _within(got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


def _mixed(x, w):
    """[N, O, 16] in float64, one product for each component."""
    x, w = x.double(), w.double()
    return torch.stack([x[:, :, m].contiguous() @ w[l] for m, l in enumerate(DEGREE)], 2)


# ---------------------------------------------------------------------------
# channel mixing with its weight in registers: tiles after the first
# ---------------------------------------------------------------------------

def _atoms(k, m):
    """So many that each workgroup takes three tiles of 16 atoms, some a fourth, with an odd end.  At
    most 512 workgroups share the atoms, for one chunk of outputs (32 or 64, above 128 channels 16 or
    32); with more chunks as many fewer."""
    outputs = 16 if k > 128 else 32
    chunks = -(-m // (outputs if m <= outputs else 2 * outputs))
    return 16 * (3 * 8 * max(1, 64 // chunks) + 5) + 11


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype,k,m", [("f32", k, m) for k in (24, 33, 64) for m in (20, 64, 200)]
                         + [("bf16", k, m) for k in (9, 64, 70, 100, 128, 130, 200, 256)
                            for m in (16, 20, 64, 130)])
def test_mixing_takes_many_tiles(dev, dtype, k, m, transposed):
    n = _atoms(k, m)
    x = _features(dev, n, k, dtype, k + m)
    w = torch.randn(4, k, m, generator=_gen(dev, 3), device=dev) / k ** 0.5
    y = _batmobile.channel_mixing(x, w.transpose(1, 2).contiguous(), True) if transposed else \
        _batmobile.channel_mixing(x, w)
    want, size = _mixed(x, w), _mixed(x.abs(), w.abs())
    more, out = (2.0 ** -15, 2.0 ** -8) if dtype == "bf16" else (0.0, 0.0)
    _within(y, want, size * ((k + 16) * U + more) + want.abs() * out)
    for _ in range(3):
        again = _batmobile.channel_mixing(x, w.transpose(1, 2).contiguous(), True) if transposed \
            else _batmobile.channel_mixing(x, w)
        assert torch.equal(again, y)


def test_the_reference_here_is_the_oracle(dev):
    from oracle import layers as ol
    x = _features(dev, 30, 5, "f32", 1)
    w = torch.randn(4, 5, 7, generator=_gen(dev, 3), device=dev)
    y = ol.channel_mixing(x.cpu().numpy(), w.cpu().numpy())
    # float64 both, sums of 5 terms in another order
    assert (_mixed(x, w).cpu() - torch.from_numpy(y)).abs().max() <= 1e-12


# ---------------------------------------------------------------------------
# launches after the first
# ---------------------------------------------------------------------------

def _rows_that_count(n, chunk):
    """The ends of launches, and of what 2^32 threads take."""
    at = sorted({0, n} | set(range(chunk, n, chunk)))
    return [slice(max(0, a - 40), min(n, a + 40)) for a in at]


@pytest.mark.parametrize("dtype,n", [("f32", (1 << 29) + 3), ("bf16", (1 << 30) + 3)])
def test_activation_and_codes_of_very_many_atoms(dev, dtype, n):
    """One channel, within the documented N ceil(C / 8) < 2^31: more than 2^32 threads in all."""
    torch.cuda.empty_cache()
    x = torch.zeros(n, 1, 16, dtype=TYPES[dtype], device=dev)
    rows = _rows_that_count(n, 1 << 27)
    for i, part in enumerate(rows):
        x[part] = _features(dev, part.stop - part.start, 1, dtype, i)
    codes, exps = _batmobile.checkpoint_encode(x)
    for part in rows:
        c, e = _batmobile.checkpoint_encode(x[part])
        assert torch.equal(codes[part].view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(exps[part], e)
    back = _batmobile.checkpoint_decode(codes, exps, TYPES[dtype])
    for part in rows:
        assert torch.equal(back[part], _batmobile.checkpoint_decode(codes[part].clone(), exps[part].clone(),
                                                                    TYPES[dtype]))
    del back
    y, c, e = _batmobile.gate_activation(x, True)
    assert torch.equal(e, exps) and torch.equal(c.view(torch.uint8), codes.view(torch.uint8))
    del c, e
    for part in rows:
        assert torch.equal(y[part], _batmobile.gate_activation(x[part])[0])
    # (the output as the gradient that comes in)
    gx = _batmobile.gate_activation_backward(y, x, None, None)
    for part in rows:
        assert torch.equal(gx[part], _batmobile.gate_activation_backward(y[part], x[part], None, None))
    del gx
    gx = _batmobile.gate_activation_backward(y, None, codes, exps)
    for part in rows:
        assert torch.equal(gx[part], _batmobile.gate_activation_backward(
            y[part], None, codes[part].clone(), exps[part].clone()))
    del x, y, gx, codes, exps
    torch.cuda.empty_cache()
