"""The operators beside attention where a workgroup goes on to further work: tiles of atoms, steps of a
range, batches of edges, launches after the first.  Every row differs from every other.

Bounds, u = 2^-24:
  mixing    a sum of K products, each as exact as one of fp32: (K + 16) u sum |x w|; bf16: the weight to
            2^-15, the result to 2^-8 of itself more
  gW        a sum of n (2 l + 1) products of exact values: (n (2 l + 1) + 16) u sum |x g|; as a whole 3e-6, as
            roundings do not add up one way
  gtable    a sum of n terms in any order: (n + 8) u sum |g|
  glengths  a sum of H terms, and six roundings of the factor: (H + 8) u sum |g| |factor|
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


def _weight_gradient(x, g):
    x, g = x.double(), g.double()
    out = torch.zeros(4, x.shape[1], g.shape[1], dtype=torch.float64, device=x.device)
    for m, l in enumerate(DEGREE):
        out[l] += x[:, :, m].t().contiguous() @ g[:, :, m].contiguous()
    return out


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
    x, g = _features(dev, 30, 5, "f32", 1), _features(dev, 30, 7, "f32", 2)
    w = torch.randn(4, 5, 7, generator=_gen(dev, 3), device=dev)
    y, _, gw = ol.channel_mixing(x.cpu().numpy(), w.cpu().numpy(), g.cpu().numpy())
    # float64 both, sums of up to 210 terms in another order
    assert (_mixed(x, w).cpu() - torch.from_numpy(y)).abs().max() <= 1e-12
    assert (_weight_gradient(x, g).cpu() - torch.from_numpy(gw)).abs().max() <= 1e-12


# ---------------------------------------------------------------------------
# the weight's gradient: steps after the first of a range of atoms
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,c,o", [(12345, 64, 64), (12295, 20, 40), (1003, 128, 1024), (2501, 70, 300),
                                   (1507, 200, 300), (1001, 1024, 65), (4101, 100, 200)])
def test_weight_gradient_takes_many_steps(dev, dtype, kept, n, c, o):
    """At most 256 workgroups take 64 or 128 channels by 64 each over ranges of steps of 16 atoms (8 in
    fp32): three steps of a range at least here, and an odd end."""
    x, g = _features(dev, n, c, dtype, c), _features(dev, n, o, dtype, o + 1)
    if kept:
        codes, exps = _batmobile.checkpoint_encode(x)
        x = _batmobile.checkpoint_decode(codes, exps, torch.float32)
        gw = _batmobile.channel_mixing_weight_grad(None, codes, exps, g)
    else:
        gw = _batmobile.channel_mixing_weight_grad(x, None, None, g)
    want, size = _weight_gradient(x, g), _weight_gradient(x.abs(), g.abs())
    terms = n * torch.tensor([1.0, 3, 5, 7], device=dev, dtype=torch.float64)[:, None, None]
    _within(gw, want, size * (terms + 16) * U)
    assert (gw - want).abs().max() <= 3e-6 * want.abs().max()


# ---------------------------------------------------------------------------
# the bias's table: batches of edges after the first of a share
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("e,b,h", [(900_001, 64, 8), (450_007, 65, 8), (450_003, 128, 8),
                                   (260_011, 200, 8), (260_005, 300, 8), (70_003, 200, 40),
                                   (40_009, 150, 64), (40_013, 300, 70), (900_009, 7, 8)])
def test_table_gradient_takes_many_batches(dev, e, b, h):
    """At most 512 workgroups share the edges; a batch is 16 steps (8 up to 64 buckets) of each wave."""
    gen = _gen(dev, b + h)
    k = torch.randint(0, b, (e,), generator=gen, device=dev)
    g = torch.randn(e, h, generator=gen, device=dev)
    gt, _ = _batmobile.distance_bias_backward(None, k.short(), g, b, 0.0, True, False)
    zero = torch.zeros(b, h, dtype=torch.float64)
    k, g = k.cpu(), g.cpu().double()
    want, size = zero.index_add(0, k, g), zero.index_add(0, k, g.abs())
    _within(gt.cpu(), want, (torch.bincount(k, minlength=b)[:, None] + 8) * U * size)
    assert (gt.cpu() - want).abs().max() <= 3e-6 * size.max()


# ---------------------------------------------------------------------------
# launches after the first
# ---------------------------------------------------------------------------

def test_lengths_gradient_takes_a_second_launch(dev):
    """A launch takes 2^26 edges with 16 lanes an edge."""
    e, h, c = (1 << 26) + 77, 9, 5.0
    gen = _gen(dev, 4)
    r, g = 6 * torch.rand(e, generator=gen, device=dev), torch.empty(e, h, device=dev)
    g.normal_(generator=gen)
    _, gl = _batmobile.distance_bias_backward(r, None, g, 1, c, False, True)
    for part in (slice(0, 500), slice((1 << 26) - 500, e)):
        q, gq = r[part].double(), g[part].double()
        factor = torch.where(q < c, -2 * q / ((c - q) * (c + q)), 0.0)
        _within(gl[part], factor * gq.sum(1), (h + 8) * U * factor.abs() * gq.abs().sum(1))


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
