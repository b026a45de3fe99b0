"""Global norm of gradients and clipping, over many tensors in two kernels.

Not a reference API.  norm = sqrt(sum over all tensors of g^2), summed in 64 bits; the
gradients become g * min(1, max_norm / (norm + 1e-6)).  Nothing waits for the GPU: the norm is
returned as a tensor.  float32 and bfloat16 tensors may be mixed.
"""
import torch

import _batmobile


def clip_grad_norm(grads, max_norm, out=None):
    """(norm, clipped): the clipped gradients in `out` (a list like grads; None: new tensors).

    out may hold grads themselves, in any order, or other tensors that share memory with them: all
    of grads is read first.  A tensor that is listed twice counts twice in the norm and is scaled
    once.
    """
    norm, clipped = _batmobile.clip_grad_norm(grads, max_norm, out)
    return norm, clipped if out is None else out


def clip_grad_norm_(parameters, max_norm):
    """Clips the gradients of `parameters` in place; returns their norm before clipping.  A
    parameter that is listed twice (tied weights) counts and is scaled once."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in dict.fromkeys(parameters) if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return clip_grad_norm(grads, max_norm, grads)[0]
