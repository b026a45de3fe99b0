"""A learned bias of attention by distance, with its gradients.

Not a reference API.  The relative position of two atoms that attention may know is their distance;
it falls into one of B buckets, each with a number for every head:

    bias[e, h] = table[number of boundaries <= r_e, h] + log(1 - (r_e / cutoff)^2)

The second term (with a cutoff) takes an edge's weight to 0 smoothly; from the cutoff on the bias
is -inf, which `neighbor_attention` leaves out.
"""
import _batmobile


def distance_bias(lengths, boundaries, table, cutoff=None):
    """bias [E, H] of lengths [E], boundaries [B - 1] ascending, table [B, H], all float32, for
    `neighbor_attention`. Up to 4096 buckets and 1024 heads; cutoff from 1e-30 to 1e30. Gradients
    for the table and, through the cutoff's term, for the lengths (0 from the cutoff on; without a
    cutoff 0 everywhere), the same from run to run; none for the boundaries, no second and no
    forward-mode derivatives (errors).
    """
    return _batmobile.distance_bias_autograd(lengths, boundaries, table,
                                             None if cutoff is None else float(cutoff))
