"""An equivariant transformer block on an atom graph, with gradients for training.

Not a reference API.  Node features [N, C, 16] (degrees 0 to 3) pass through

    n  = norm(x; norm)                                   (given by the block before, if any)
    q, k, v = channel mixing of n, degree by degree      (k, v: kv_heads of the heads' size)
    b_eh = MLP(basis(r_e))_h + log envelope(r_e)         (-inf at the cutoff: the edge ends)
    a  = attention of every atom over its neighbours     (neighbor_attention)
    y  = channel mixing of a, gate = linear(scalars of n)
    h  = x + scale sigmoid(gate) norm(y; norm_post),  n' = norm(h; next norm)

A head is heads' share of the channels with all their components, whose products do not change
under rotations, so the block commutes with them.  The mixings are plain matrix products of the
caller's torch; everything else runs in the HIP kernels.  The edge lengths come from the graph
as numbers: gradients reach the features and the parameters, not the positions, so a model of this
block alone has no forces (MACEInteraction gives those).
"""
import math

import torch

from .attention import neighbor_attention
from .block_norm import equivariant_norm, gated_residual_norm

N_BASIS = 8
HIDDEN = 32


def _mix(x, weight):
    """Channels of each degree by weight [4, C_in, C_out]: [N, C_in, 16] -> [N, C_out, 16]."""
    n, c = x.shape[:2]
    x = x.transpose(1, 2)                                # [N, 16, C]
    parts = []
    for l in range(4):
        rows = x[:, l * l:(l + 1) ** 2].reshape(-1, c)   # a copy: components of degree l
        parts.append((rows @ weight[l].to(x.dtype)).view(n, 2 * l + 1, -1))
    return torch.cat(parts, 1).transpose(1, 2).contiguous()


class AttentionBlock(torch.nn.Module):
    """channels must be a multiple of heads, heads one of kv_heads, and channels / heads at most
    16 (head size 256).  Parameters are float32; features may be float32 or bfloat16."""

    def __init__(self, channels, heads, kv_heads=None, cutoff=5.0, device=None, generator=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads or channels // heads > 16:
            raise ValueError("AttentionBlock: channels must be a multiple of heads (at most 16 "
                             "each) and heads one of kv_heads")
        self.channels, self.heads, self.kv_heads = channels, heads, kv_heads
        self.cutoff = float(cutoff)
        self.kv_channels = channels // heads * kv_heads
        g = generator

        def normal(*shape):
            w = torch.randn(*shape, generator=g) / math.sqrt(shape[-2])
            return torch.nn.Parameter(w.to(device))

        self.norm = torch.nn.Parameter(torch.ones(4, channels, device=device))
        self.norm_post = torch.nn.Parameter(torch.ones(4, channels, device=device))
        self.scale = torch.nn.Parameter(torch.full((channels,), 0.5, device=device))
        self.w_qkv = normal(4, channels, channels + 2 * self.kv_channels)
        self.w_out = normal(4, channels, channels)
        self.w_gate = normal(channels, 4 * channels)
        self.w1, self.w2 = normal(N_BASIS, HIDDEN), normal(HIDDEN, heads)

    def edge_bias(self, lengths):
        """[E, H]: a function of the edge length, -inf from the cutoff on."""
        d = (lengths / self.cutoff).clamp(max=1.0)
        k = torch.arange(1, N_BASIS + 1, device=lengths.device, dtype=lengths.dtype)
        basis = torch.sinc(k * d[:, None])
        envelope = torch.log((1 - d * d).clamp(min=0))
        return torch.nn.functional.silu(basis @ self.w1) @ self.w2 + envelope[:, None]

    def forward(self, graph, x, n=None, next_norm=None):
        """graph: batmobile.Graph; x [N, C, 16]; n: norm(x; self.norm) where the block before
        has formed it; next_norm: the norm weight of the block behind.  Returns (h, n') or,
        without next_norm, h."""
        if n is None:
            n = equivariant_norm(x, self.norm)
        atoms, c, kv = x.shape[0], self.channels, self.kv_channels
        size = c // self.heads * 16
        q, k, v = _mix(n, self.w_qkv).split([c, kv, kv], 1)
        bias = self.edge_bias(graph.exact().vec.norm(dim=1))
        a = neighbor_attention(q.reshape(atoms, self.heads, size),
                               k.reshape(atoms, self.kv_heads, size),
                               v.reshape(atoms, self.kv_heads, size), graph.attention_plan(),
                               bias=bias)
        y = _mix(a.view(atoms, c, 16), self.w_out)
        gate = (n[:, :, 0].contiguous() @ self.w_gate.to(n.dtype)).view(atoms, c, 4)
        return gated_residual_norm(x, y, gate, self.scale, self.norm_post, next_norm)
