"""Softmax attention over the edges of a graph, with gradients.

Not a reference API (the reference sums its messages).  For every destination i and head h,
over the edges e: j -> i of the graph,

    x_eh = scale <q[i, h], k[j, g]> + bias[e, h],  p = softmax over the row,
    out[i, h] = sum_e p_eh v[j, g],                g = h // (H / H_kv)

Equivariant features [N, C, 16] go in as heads of C / H channels, `x.view(N, H, C // H * 16)`:
the product over a channel's 16 components does not change under rotations.  The backward
recomputes the probabilities from each row's reference and sum; no sum's order varies, so results
are the same from run to run.
"""
import math

import torch

import _batmobile


class AttentionPlan:
    """The edges of a graph as the attention kernels take them, made once per graph.

    src [E] int64 are the sources in the order of row_ptr [n_dst + 1] (edges grouped by
    destination), ascending within a row.  order and src_order are permutations of the
    destinations and of the sources: 16 that follow each other form a tile, whose shared
    neighbours are read once, so spatially near ones should be next to each other
    (`spatial_order`); results only differ in the order of summation.  from_edge_index takes
    edges in any order; bias rows are always in the caller's order of the edges.  Making a plan
    waits for the GPU once.  validate=False leaves out the check of the arrays (the kernels then
    rely on them).
    """

    def __init__(self, src, row_ptr, n_src=None, order=None, src_order=None, edge_id=None,
                 validate=True, _sorted_here=False):
        for name, t in (("src", src), ("row_ptr", row_ptr), ("order", order),
                        ("src_order", src_order), ("edge_id", edge_id)):
            if t is None and name not in ("src", "row_ptr"):
                continue
            if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous():
                raise ValueError(f"AttentionPlan: {name} must be a contiguous int64 vector")
            if t.device != src.device:
                raise ValueError(f"AttentionPlan: {name} must be on the device of src")
        self.src, self.row_ptr = src, row_ptr
        self.n_dst = row_ptr.numel() - 1
        self.n_src = self.n_dst if n_src is None else int(n_src)
        self.edge_id = None if edge_id is None else edge_id.int()
        self._src_order, self._source_side = src_order, None
        if validate:
            for name, t, n in (("order", order, self.n_dst), ("src_order", src_order, self.n_src),
                               ("edge_id", None if _sorted_here else edge_id, src.numel())):
                if t is not None and not torch.equal(t.sort()[0],
                                                     torch.arange(n, device=t.device)):
                    raise ValueError(f"AttentionPlan: {name} must be a permutation")
        # last: it waits for the stream, so that any stream may use the plan from here on
        plan, items, parts, bad = _batmobile.attention_plan(row_ptr, src, order, self.n_src,
                                                            validate)
        if bad & 1 or (self.n_dst == 0 and src.numel()):
            raise ValueError("AttentionPlan: row_ptr must rise from 0 to the number of edges")
        if bad & 2:
            raise ValueError(f"AttentionPlan: src must lie in [0, {self.n_src})")
        if bad & 4:
            raise ValueError("AttentionPlan: src must ascend within a row (from_edge_index takes "
                             "edges in any order)")
        if bad & 8:
            raise ValueError("AttentionPlan: row_ptr and order give the rows more edges than there "
                             "are")
        self.side = (plan, items, parts)

    @classmethod
    def from_edge_index(cls, edge_index, n_dst, n_src=None, order=None, src_order=None):
        """edge_index [2, E] (sources, destinations) in any order."""
        if edge_index.dim() != 2 or edge_index.shape[0] != 2:
            raise ValueError("AttentionPlan: edge_index must be [2, E]")
        n_src = n_dst if n_src is None else n_src
        src, dst = edge_index[0], edge_index[1]
        if dst.numel() and not bool(((dst >= 0) & (dst < n_dst)).all()):
            raise ValueError(f"AttentionPlan: destinations must lie in [0, {n_dst})")
        edge_id = torch.argsort(dst * n_src + src, stable=True)
        rows = torch.arange(n_dst + 1, device=dst.device)
        row_ptr = torch.searchsorted(dst[edge_id], rows)
        # (argsort's edge_id is a permutation as it comes, so not checked)
        return cls(src[edge_id], row_ptr, n_src, order, src_order, edge_id, _sorted_here=True)

    def source_side(self):
        """The edges grouped by source, for the backward (built when gradients are first wanted):
        the side's plan and the place of every edge in its order."""
        if self._source_side is None:
            dst = torch.repeat_interleave(
                torch.arange(self.n_dst, device=self.src.device), self.row_ptr.diff(),
                output_size=self.src.numel())
            by, pos = torch.sort(self.src, stable=True)
            rows = torch.arange(self.n_src + 1, device=self.src.device)
            place = torch.empty_like(pos, dtype=torch.int32)
            place[pos] = torch.arange(pos.numel(), dtype=torch.int32, device=pos.device)
            # last: it waits for the stream, so that any stream may use the result from here on
            plan, items, parts, bad = _batmobile.attention_plan(
                torch.searchsorted(by, rows), dst[pos], self._src_order, self.n_dst, False)
            if bad:
                raise ValueError("AttentionPlan: src_order must be a permutation")
            self._source_side = (plan, items, parts, place)
        return self._source_side


def neighbor_attention(q, k, v, plan, bias=None, scale=None):
    """Attention of each destination over its edges: out [n_dst, H, Dv].

    q [n_dst, H, Dk], k [n_src, H_kv, Dk], v [n_src, H_kv, Dv] in float32 or bfloat16 (sums and
    softmax in float32), H a multiple of H_kv, Dk and Dv up to 256; rows may be strided (slices
    of one projection).  bias [E, H] float32: an edge with -inf is left out.  A row without an
    edge gives zeros.  scale defaults to 1 / sqrt(Dk).  Gradients for q, k, v and bias,
    which cannot be differentiated again, and no forward-mode derivatives (an error, not a
    missing term).
    """
    if q.dim() == 3 and (q.shape[0] != plan.n_dst or k.shape[0] != plan.n_src):
        raise RuntimeError(f"neighbor_attention: the plan has {plan.n_dst} destinations and "
                           f"{plan.n_src} sources")
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    return _batmobile.neighbor_attention_autograd(q, k, v, bias, *plan.side, plan.src.numel(),
                                                  plan.edge_id, plan.row_ptr, plan.source_side,
                                                  scale)
