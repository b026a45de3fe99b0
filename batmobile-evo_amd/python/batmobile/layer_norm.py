"""Layer norm of invariant features, with gradients.

Not a reference API.  The mean may be taken off only where rotations change nothing: hidden features
of edges, or the invariants x[:, :, 0] of features [N, C, 16], which are read where they lie.
"""
import _batmobile


def layer_norm(x, weight, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x [..., D].

    x float32 or bfloat16 at any strides (rows at one stride are read in place), D up to 8192;
    weight and bias [D] float32, sums in float32.  Gradients for x, weight and bias, the same from run
    to run, which cannot be differentiated again, and no forward-mode derivatives (an error).
    """
    return _batmobile.layer_norm_autograd(x, weight, bias, float(eps))
