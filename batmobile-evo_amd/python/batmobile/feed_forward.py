"""Channel mixing, the gated activation and the feed-forward block, with 8-bit checkpoints.

Not a reference API.  Features [N, C, 16] hold the components of degrees 0 to 3 of C channels;
what mixes channels within a degree, or scales all components of one, commutes with rotations:

    channel_mixing:   y[o, m] = sum_c x[c, m] W[l(m), c, o]
    gate_activation:  y[c, m] = sigmoid(x[c, 0]) x[c, m]        (silu of the invariant)

With checkpoint="e4m3" a layer keeps its input for the backward pass in 8 bits instead of 16 or 32:
blocks of 8 channels of an atom share a power of two, the least with max |x| <= 448 times it (2^-110
to 2^120), and hold x over it as e4m3: a value is off by 2^-4 of itself at most, one below 2^-6
times the power (2^-13.8 of the block's largest) by 2^-10 times the power. The output and what the
gradient passes on through a mixing do not change; the weight's gradient, and the activation's, are
those at the input so kept. A value that is not finite is kept as NaN.
"""
import math

import torch

import _batmobile

from .block_norm import equivariant_norm, gated_residual_norm
from .layer_norm import layer_norm


def channel_mixing(x, weight, checkpoint=None):
    """y [N, C_out, 16] of x [N, C_in, 16] (float32 or bfloat16) and weight [4, C_in, C_out]
    (float32), up to 2048 channels.  float32 features have float32 accuracy (numbers below 2^-110
    only that of 2^-133); with bfloat16 ones the weight is taken to 15 bits and sums are float32,
    which leaves the error of the result's own rounding.  Gradients for both, which cannot be
    differentiated again, and no forward-mode derivatives (an error).  checkpoint: None, or "e4m3",
    with which an infinite float32 gradient makes its column of the weight's gradient NaN.
    """
    return _batmobile.channel_mixing_autograd(x, weight, checkpoint)


def gate_activation(x, checkpoint=None):
    """sigmoid(x[:, :, :1]) * x of x [N, C, 16] (float32 or bfloat16), up to 2048 channels.  One
    gradient, which cannot be differentiated again, and no forward-mode derivatives (an error).
    checkpoint: None, or "e4m3"."""
    return _batmobile.gate_activation_autograd(x, checkpoint)


def checkpoint_encode(x):
    """(codes [N, C, 16] float8_e4m3fn, exponents [N, ceil(C / 8)] uint8) of x [N, C, 16]: the 8-bit
    form as the layers keep it, for a caller's own autograd functions.  Has no gradient."""
    return _batmobile.checkpoint_encode(x.detach())


def checkpoint_decode(codes, exponents, dtype=torch.float32):
    """The features that checkpoint_encode's result holds: codes * 2^(exponents - 127)."""
    return _batmobile.checkpoint_decode(codes, exponents, dtype)


class FeedForwardBlock(torch.nn.Module):
    """The half of a transformer block that AttentionBlock leaves to it:

        n = norm(x; norm)                                       (given by the block before, if any)
        y = channel_mixing(gate_activation(channel_mixing(n, w1)), w2)
        gate = linear(layer_norm(invariants of x))
        h = x + scale sigmoid(gate) norm(y; norm_post),  n' = norm(h; next norm)

    hidden: channels between the mixings (default 2 channels).  checkpoint="e4m3" keeps the mixings'
    and the activation's inputs in 8 bits while training.  Parameters are float32; features may be
    float32 or bfloat16.
    """

    def __init__(self, channels, hidden=None, checkpoint=None, device=None, generator=None):
        super().__init__()
        hidden = 2 * channels if hidden is None else hidden
        if checkpoint not in (None, "e4m3"):
            raise ValueError('FeedForwardBlock: checkpoint must be None or "e4m3"')
        self.channels, self.hidden, self.checkpoint = channels, hidden, checkpoint

        def normal(*shape):
            w = torch.randn(*shape, generator=generator) / math.sqrt(shape[-2])
            return torch.nn.Parameter(w.to(device))

        self.norm = torch.nn.Parameter(torch.ones(4, channels, device=device))
        self.norm_post = torch.nn.Parameter(torch.ones(4, channels, device=device))
        self.scale = torch.nn.Parameter(torch.full((channels,), 0.5, device=device))
        self.gate_norm = torch.nn.Parameter(torch.ones(channels, device=device))
        self.gate_shift = torch.nn.Parameter(torch.zeros(channels, device=device))
        self.w1, self.w2 = normal(4, channels, hidden), normal(4, hidden, channels)
        self.w_gate = normal(channels, 4 * channels)

    def forward(self, x, n=None, next_norm=None):
        """x [N, C, 16]; n: norm(x; self.norm) where the block before has formed it; next_norm: the
        norm weight of the block behind.  Returns (h, n') or, without next_norm, h."""
        if n is None:
            n = equivariant_norm(x, self.norm)
        u = channel_mixing(n, self.w1, self.checkpoint)
        y = channel_mixing(gate_activation(u, self.checkpoint), self.w2, self.checkpoint)
        s = layer_norm(x[:, :, 0], self.gate_norm, self.gate_shift)
        gate = (s @ self.w_gate.to(s.dtype)).view(x.shape[0], self.channels, 4)
        return gated_residual_norm(x, y, gate, self.scale, self.norm_post, next_norm)
