"""Norms by degree of equivariant features, alone and fused with the end of a block.

Not a reference API.  Features [N, C, 16] hold the components of degrees 0 to 3 of C channels;
every degree l of an atom is divided by its root mean square over channels and components:

    norm(z; w)[c, lm] = w[l, c] z[c, lm] / sqrt(mean z_l^2 + eps)

float32 or bfloat16 features, float32 weights and sums, one pass over the data each way.
"""
import torch
from torch.autograd.function import once_differentiable

import _batmobile


class GatedResidualNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, scale, weight_post, weight_pre, eps):
        train = any(ctx.needs_input_grad[:6])
        h, n, rs = _batmobile.gated_residual_norm(x, y, gate, scale, weight_post, weight_pre,
                                                  eps, train)
        ctx.save_for_backward(x, y, gate, scale, weight_post, weight_pre, rs)
        ctx.set_materialize_grads(False)
        if y is None:
            return n
        return h if n is None else (h, n)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x, y, gate, scale, weight_post, weight_pre, rs = ctx.saved_tensors
        if all(g is None for g in grads):
            return (None,) * 7
        gh = None if y is None else grads[0]
        gn = None if weight_pre is None else grads[-1]
        if gn is None:          # only h is used further on
            weight_pre_used, gw_zero = None, weight_pre is not None
        else:
            weight_pre_used, gw_zero = weight_pre, False
        gx, gy, gg, gs, gpost, gpre = _batmobile.gated_residual_norm_backward(
            gh, gn, x, y, gate, scale, weight_post, weight_pre_used, rs)
        if gw_zero:
            gpre = torch.zeros_like(weight_pre)
        return gx, gy, gg, gs, gpost, gpre, None


def equivariant_norm(x, weight, eps=1e-6):
    """norm(x; weight) of x [N, C, 16], weight [4, C] (before a block)."""
    return GatedResidualNormFunction.apply(x, None, None, None, None, weight, float(eps))


def gated_residual_norm(x, y, gate, scale, weight_post, weight_pre=None, eps=1e-6):
    """The end of a block and the start of the next, in one kernel:

        h = x + scale[c] sigmoid(gate[c, l]) norm(y; weight_post),  n = norm(h; weight_pre)

    x (residual), y (the block's output) [N, C, 16], gate [N, C, 4] (None: no gate), scale [C],
    weights [4, C].  Returns (h, n), or h where weight_pre is None (after the last block).
    Gradients for every tensor, which cannot be differentiated again (an error).
    """
    return GatedResidualNormFunction.apply(x, y, gate, scale, weight_post, weight_pre, float(eps))
