"""The operators beside attention together: the feed-forward block and the attention block's learned
table and 8-bit checkpoints, against a float64 composition, under rotations, and as training steps."""
import numpy as np
import pytest
import torch

from oracle import block as ob
from oracle import layers as ol

from helpers import gen, normwise_err, periodic_box, random_rotation, wigner_d

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().cpu().double().numpy()


def _graph(dev, n, seed, channels):
    import batmobile
    pos, cell = periodic_box(n, seed)
    return batmobile.Graph(pos.to(dev), cell, 5.0, channels)


def _feed_forward(block, x, next_norm):
    """The block from the float64 oracle's operators."""
    p = {k: _np(v) for k, v in block.named_parameters()}
    n = ob.norm(x, p["norm"])[0]
    y = ol.channel_mixing(ol.gate_activation(ol.channel_mixing(n, p["w1"])), p["w2"])
    s = ol.layer_norm(x[:, :, 0], p["gate_norm"], p["gate_shift"])
    gate = (s @ p["w_gate"]).reshape(x.shape[0], x.shape[1], 4)
    return ob.gated_residual_norm(x, y, gate, p["scale"], p["norm_post"], next_norm)


@pytest.mark.parametrize("c,hidden", [(16, None), (20, 33), (8, 8)])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_feed_forward_against_float64(dev, c, hidden, checkpoint):
    """Bound: six operators and a matrix product of fp32 in a row, 1e-5 each at most: 7e-5.  What the
    forward gives does not depend on how the inputs are kept."""
    import batmobile
    block = batmobile.FeedForwardBlock(c, hidden, checkpoint, dev, gen(1))
    with torch.no_grad():
        block.gate_shift.copy_(torch.randn(c, generator=gen(2)))
    x = torch.randn(90, c, 16, generator=gen(3))
    w = torch.rand(4, c, generator=gen(4)) + 0.5
    h, n = block(x.to(dev), next_norm=w.to(dev))
    want = _feed_forward(block, x.double().numpy(), w.double().numpy())
    assert normwise_err(_np(h), want[0]) <= 7e-5 and normwise_err(_np(n), want[1]) <= 7e-5


def test_feed_forward_gradients_against_differences(dev):
    """Along a random direction of all parameters and features, by central differences of the float64
    composition.  fp32 gradients, 1e-4 of the slope's terms; the differences' own error is h^2."""
    import batmobile
    block = batmobile.FeedForwardBlock(12, 20, None, dev, gen(5))
    x = torch.randn(30, 12, 16, generator=gen(6)).to(dev).requires_grad_(True)
    g = torch.randn(30, 12, 16, generator=gen(7)).to(dev)
    leaves = [x] + list(block.parameters())
    grads = torch.autograd.grad(block(x), leaves, g)
    step = [torch.randn(t.shape, generator=gen(8 + i)).double() for i, t in enumerate(leaves)]
    slope = sum(float((a.cpu().double() * b).sum()) for a, b in zip(grads, step))
    size = sum(float((a.cpu().double() * b).norm()) for a, b in zip(grads, step))
    h = 1e-5

    class Moved:
        def __init__(self, k):
            self.k = k

        def named_parameters(self):
            return [(n, p.detach().cpu().double() + self.k * h * s)
                    for (n, p), s in zip(block.named_parameters(), step[1:])]

    def value(k):
        out = _feed_forward(Moved(k), _np(x) + k * h * step[0].numpy(), None)[0]
        return (out * _np(g)).sum()

    assert abs((value(1) - value(-1)) / (2 * h) - slope) <= 1e-4 * size


def test_feed_forward_commutes_with_rotations(dev):
    import batmobile
    block = batmobile.FeedForwardBlock(16, 24, None, dev, gen(20))
    x = torch.randn(70, 16, 16, generator=gen(21))
    d = torch.from_numpy(wigner_d(random_rotation(7)))
    a, b = block(x.to(dev)), block((x.double() @ d.T).float().to(dev))
    assert normwise_err(_np(b), _np(a) @ d.T.numpy()) <= 5e-5


def test_checkpoints_change_the_weights_gradients_alone_through_a_mixing(dev):
    """With w2 alone trained, its gradient is that at the kept input; that of one mixing's input is
    the same either way."""
    import batmobile
    x = torch.randn(50, 12, 16, generator=gen(22)).to(dev).requires_grad_(True)
    w = torch.randn(4, 12, 9, generator=gen(23)).to(dev).requires_grad_(True)
    g = torch.randn(50, 9, 16, generator=gen(24)).to(dev)
    a = torch.autograd.grad(batmobile.channel_mixing(x, w), [x, w], g)
    b = torch.autograd.grad(batmobile.channel_mixing(x, w, "e4m3"), [x, w], g)
    assert torch.equal(a[0], b[0])
    kept = batmobile.checkpoint_decode(*batmobile.checkpoint_encode(x))
    c, = torch.autograd.grad(batmobile.channel_mixing(kept, w), w, g)
    assert normwise_err(_np(b[1]), _np(c)) <= 1e-6
    # the codes are off by 2^-4 of a value at most, independently: far less in a sum of 50 to 350
    assert 0 < normwise_err(_np(b[1]), _np(a[1])) <= 2.0 ** -4


@pytest.mark.parametrize("target", [False, True])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_steps_of_a_transformer(dev, dtype, checkpoint, target):
    """Attention with a learned table and feed-forward, two of each, norms handed on: every parameter
    gets a finite gradient, and the clipped norm is the limit times norm / (norm + 1e-6), by the
    clipping's definition (without a target the loss is of normed values, nearly constant, and the
    gradients are small against 1e-6)."""
    import batmobile
    c = 32
    graph = _graph(dev, 200, 30, c)
    model = torch.nn.ModuleList()
    for k in range(2):
        model.append(batmobile.AttentionBlock(c, 4, 2, device=dev, generator=gen(31 + k), buckets=24,
                                              checkpoint=checkpoint))
        model.append(batmobile.FeedForwardBlock(c, 48, checkpoint, dev, gen(41 + k)))
    x = torch.randn(200, c, 16, generator=gen(51)).to(dev, dtype)
    want = torch.randn(200, c, 16, generator=gen(52)).to(dev)
    last = torch.ones(4, c, device=dev)
    for _ in range(3):
        h, n = x, batmobile.equivariant_norm(x, model[0].norm)
        for k, block in enumerate(model):
            norm = model[k + 1].norm if k < 3 else last
            h, n = block(graph, h, n, norm) if k % 2 == 0 else block(h, n, norm)
        (n.float() - want if target else n.float()).square().mean().backward()
        for name, p in model.named_parameters():
            assert p.grad is not None and torch.isfinite(p.grad).all(), name
        total = float(torch.cat([p.grad.flatten() for p in model.parameters()]).double().norm())
        limit = 0.5 * total
        batmobile.clip_grad_norm_(model.parameters(), limit)
        clipped = float(torch.cat([p.grad.flatten() for p in model.parameters()]).double().norm())
        assert total > 0 and abs(clipped - limit * total / (total + 1e-6)) <= 1e-5 * limit
        with torch.no_grad():
            for p in model.parameters():
                p -= 0.1 * p.grad
                p.grad = None


def test_attention_block_with_a_table(dev):
    """The bias of the block is the table's, next to the same block with the bias formed by hand."""
    import batmobile
    c = 16
    graph = _graph(dev, 150, 61, c)
    block = batmobile.AttentionBlock(c, 4, device=dev, generator=gen(62), buckets=16)
    lengths = graph.exact().vec.norm(dim=1)
    bias = block.edge_bias(lengths)
    want = ol.distance_bias(_np(lengths), _np(block.boundaries), _np(block.table), block.cutoff)
    got = _np(bias)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got))
    assert np.abs(got - np.where(fine, want, 0))[fine].max() <= 1e-6 * np.abs(want[fine]).max()
    x = torch.randn(150, c, 16, generator=gen(63)).to(dev)
    out = block(graph, x)
    out.square().sum().backward()
    assert torch.isfinite(out).all() and block.table.grad.abs().sum() > 0
    assert not [n for n, p in block.named_parameters() if p.grad is None]


def test_attention_block_keeps_its_results_with_checkpoints(dev):
    """Mixings in the kernel instead of torch's products: fp32 roundings of both, 5e-5 through the
    block."""
    import batmobile
    c = 32
    graph = _graph(dev, 150, 71, c)
    a = batmobile.AttentionBlock(c, 4, device=dev, generator=gen(72))
    b = batmobile.AttentionBlock(c, 4, device=dev, generator=gen(72), checkpoint="e4m3")
    x = torch.randn(150, c, 16, generator=gen(73)).to(dev)
    assert normwise_err(_np(b(graph, x)), _np(a(graph, x))) <= 5e-5


def test_forces_through_the_cutoff(dev):
    """Lengths that depend on positions get the gradient of the bias's cutoff term: against differences
    of the float64 oracle."""
    import batmobile
    pos = torch.tensor([[0.0, 0, 0], [1.1, 0.3, 0], [0.2, 1.7, 0.5], [-1.0, 0.4, 1.2]])
    src, dst = torch.tensor([1, 2, 3, 0, 2]), torch.tensor([0, 0, 0, 1, 1])
    bound, table = torch.tensor([1.0, 1.5]), torch.randn(3, 2, generator=gen(80))
    g = torch.randn(5, 2, generator=gen(81))
    p = pos.to(dev).requires_grad_(True)
    r = (p[dst.to(dev)] - p[src.to(dev)]).norm(dim=1)
    grad, = torch.autograd.grad(batmobile.distance_bias(r, bound.to(dev), table.to(dev), 3.0), p,
                                g.to(dev))

    def value(q):
        d = np.linalg.norm(q[dst] - q[src], axis=1)
        k = (bound.numpy()[None] <= d[:, None]).sum(1)
        return ((table.numpy()[k] + np.log(1 - (d / 3.0) ** 2)[:, None]) * g.numpy()).sum()

    q, h = pos.double().numpy(), 1e-6
    for i in np.ndindex(4, 3):
        a, b = q.copy(), q.copy()
        a[i] += h
        b[i] -= h
        assert abs((value(a) - value(b)) / (2 * h) - float(grad[i])) <= 1e-5
