"""Norms by degree of equivariant features, alone and fused with the end of a block.

Not a reference API.  Features [N, C, 16] hold the components of degrees 0 to 3 of C channels;
every degree l of an atom is divided by its root mean square over channels and components:

    norm(z; w)[c, lm] = w[l, c] z[c, lm] / sqrt(mean z_l^2 + eps)

float32 or bfloat16 features, float32 weights and sums, one pass over the data each way.
"""
import _batmobile


def equivariant_norm(x, weight, eps=1e-6):
    """norm(x; weight) of x [N, C, 16], weight [4, C] (before a block)."""
    return _batmobile.gated_residual_norm_autograd(x, None, None, None, None, weight,
                                                   float(eps))[0]


def gated_residual_norm(x, y, gate, scale, weight_post, weight_pre=None, eps=1e-6):
    """The end of a block and the start of the next, in one kernel:

        h = x + scale[c] sigmoid(gate[c, l]) norm(y; weight_post),  n = norm(h; weight_pre)

    x (residual), y (the block's output) [N, C, 16], gate [N, C, 4] (None: no gate), scale [C],
    weights [4, C].  Returns (h, n), or h where weight_pre is None (after the last block).
    Gradients for every tensor, which cannot be differentiated again, and no forward-mode
    derivatives (an error).
    """
    res = _batmobile.gated_residual_norm_autograd(x, y, gate, scale, weight_post, weight_pre,
                                                  float(eps))
    return tuple(res) if len(res) == 2 else res[0]
