"""The operators beside attention where a workgroup goes on to further work: tiles of atoms, steps of a
range, batches of edges, launches after the first.  Every row differs from every other.
"""
import pytest
import torch

import _batmobile

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _features(dev, n, c, dtype, seed):
    g = _gen(dev, seed)
    return (torch.randn(n, c, 16, generator=g, device=dev)
            * torch.exp(0.5 * torch.randn(n, 1, 1, generator=g, device=dev))).to(TYPES[dtype])


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
