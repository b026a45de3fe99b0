"""The transformer block's operators together: against a float64 composition, under rotations,
and as training steps with clipped gradients."""
import numpy as np
import pytest
import torch

from oracle import block as ob

from helpers import gen, normwise_err, periodic_box, random_rotation, wigner_d

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().cpu().double().numpy()


def _graph(dev, n, seed, channels):
    import batmobile
    pos, cell = periodic_box(n, seed)
    return batmobile.Graph(pos.to(dev), cell, 5.0, channels)


def _mix(x, w):
    return np.concatenate([np.einsum("ncm,cd->ndm", x[:, :, l * l:(l + 1) ** 2], w[l])
                           for l in range(4)], 2)


def _oracle(block, graph, x, next_norm):
    """The block from the float64 oracle's operators."""
    p = {k: _np(v) for k, v in block.named_parameters()}
    n = ob.norm(x, p["norm"])[0]
    atoms, c, kv = x.shape[0], block.channels, block.kv_channels
    size = c // block.heads * 16
    q, k, v = np.split(_mix(n, p["w_qkv"]), [c, c + kv], 1)
    d = np.minimum(np.linalg.norm(_np(graph.vec), axis=1) / block.cutoff, 1.0)
    basis = np.sinc(np.arange(1, 9) * d[:, None])
    z = basis @ p["w1"]
    with np.errstate(divide="ignore"):
        bias = (z / (1 + np.exp(-z))) @ p["w2"] + np.log(np.maximum(1 - d * d, 0))[:, None]
    a = ob.attention(q.reshape(atoms, block.heads, size), k.reshape(atoms, -1, size),
                     v.reshape(atoms, -1, size), graph.src.cpu().numpy(),
                     graph.row_ptr.cpu().numpy(), bias)
    gate = (n[:, :, 0] @ p["w_gate"]).reshape(atoms, c, 4)
    return ob.gated_residual_norm(x, _mix(a.reshape(atoms, c, 16), p["w_out"]), gate, p["scale"],
                                  p["norm_post"], next_norm)


@pytest.mark.parametrize("c,h,kv", [(16, 4, 4), (32, 4, 2), (16, 1, 1)])
def test_block_against_float64(dev, c, h, kv):
    """Bound: five operators and two matrix products of fp32 in a row, 1e-5 each at most: 5e-5."""
    import batmobile
    graph = _graph(dev, 150, 61, c)
    block = batmobile.AttentionBlock(c, h, kv, device=dev, generator=gen(62))
    x = torch.randn(150, c, 16, generator=gen(63))
    w = torch.rand(4, c, generator=gen(64)) + 0.5
    out, n = block(graph, x.to(dev), next_norm=w.to(dev))
    want = _oracle(block, graph, x.double().numpy(), w.double().numpy())
    assert normwise_err(_np(out), want[0]) <= 5e-5
    assert normwise_err(_np(n), want[1]) <= 5e-5


def test_block_commutes_with_rotations(dev):
    """Features turned by D: the graph's lengths are the same, the output turns by D."""
    import batmobile
    c = 16
    graph = _graph(dev, 200, 65, c)
    block = batmobile.AttentionBlock(c, 2, device=dev, generator=gen(66))
    x = torch.randn(200, c, 16, generator=gen(67))
    d = torch.from_numpy(wigner_d(random_rotation(5)))
    a = block(graph, x.to(dev))
    b = block(graph, (x.double() @ d.T).float().to(dev))
    assert normwise_err(_np(b), _np(a) @ d.T.numpy()) <= 5e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_steps(dev, dtype):
    """Two blocks, the second fed by the first's fused norm; every parameter gets a gradient, the
    clipped norm is the limit, and the loss falls."""
    import batmobile
    c = 32
    graph = _graph(dev, 300, 68, c)
    blocks = torch.nn.ModuleList(
        [batmobile.AttentionBlock(c, 4, kv, device=dev, generator=gen(69 + kv)) for kv in (4, 2)])
    x = torch.randn(300, c, 16, generator=gen(71)).to(dev, dtype)
    target = torch.randn(300, c, 16, generator=gen(72)).to(dev)
    losses, limit = [], 0.5
    for _ in range(8):
        h, n = blocks[0](graph, x, next_norm=blocks[1].norm)
        out = blocks[1](graph, h, n)
        loss = (out.float() - target).square().mean()
        loss.backward()
        norm = batmobile.clip_grad_norm_(blocks.parameters(), limit)
        clipped = torch.cat([p.grad.flatten() for p in blocks.parameters()
                             if p.grad is not None]).double().norm()
        assert float(clipped) <= limit * 1.000001
        if float(norm) > limit:
            assert float(clipped) >= limit * 0.9999
        with torch.no_grad():
            for name, p in blocks.named_parameters():
                if name == "0.norm" or p.grad is not None:
                    assert p.grad is not None and torch.isfinite(p.grad).all(), name
                    p -= 0.5 * p.grad
                    p.grad = None
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]


def test_block_refusals(dev):
    import batmobile
    with pytest.raises(ValueError, match="multiple"):
        batmobile.AttentionBlock(30, 4)
    with pytest.raises(ValueError, match="multiple"):
        batmobile.AttentionBlock(64, 2)
    with pytest.raises(ValueError, match="multiple"):
        batmobile.AttentionBlock(32, 4, 3)


def test_block_trains_on_a_graph_of_an_evaluation_pass(dev):
    import batmobile
    block = batmobile.AttentionBlock(16, 2, device=dev, generator=gen(73))
    x = torch.randn(120, 16, 16, generator=gen(74)).to(dev)
    with torch.inference_mode():
        graph = _graph(dev, 120, 75, 16)
        want = block(graph, x)
    out = block(graph, x)
    assert torch.equal(out, want)
    out.square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in block.parameters())
