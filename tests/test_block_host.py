"""Attention, norms and clipping without a GPU: what is refused on the host before anything runs,
and the order of work around a plan's wait."""
import ctypes
import os
import types

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class _Ops(TorchDispatchMode):
    """The torch operators that run, in order."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.fixture
def plan_wait(monkeypatch):
    """(log of torch operators, their number at each wait for the GPU): attention_plan waits."""
    from batmobile import attention
    log, waits = _Ops(), []

    def attention_plan(row_ptr, col, order, n_cols, check):
        plan = torch.zeros(0, dtype=torch.int32)
        waits.append(len(log.names))
        return plan, 0, 0, 0

    monkeypatch.setattr(attention, "_batmobile",
                        types.SimpleNamespace(attention_plan=attention_plan))
    return log, waits


def test_a_plan_is_complete_when_its_constructor_returns(plan_wait):
    """Any stream may use a plan: nothing is left to run behind the wait that ends its making."""
    from batmobile import AttentionPlan
    log, waits = plan_wait
    src, dst = torch.tensor([2, 0, 1, 1, 0]), torch.tensor([1, 0, 1, 0, 1])
    with log:
        plan = AttentionPlan.from_edge_index(torch.stack([src, dst]), 2, 3)
        assert log.names[waits[-1]:] == []
        assert plan.edge_id.tolist() == [1, 3, 4, 2, 0] and plan.edge_id.dtype == torch.int32
        made = len(log.names)
        plan.source_side()
        assert len(log.names) > made and log.names[waits[-1]:] == []
        AttentionPlan(plan.src, plan.row_ptr, 3, edge_id=torch.arange(5).flip(0))
        assert log.names[waits[-1]:] == []
    assert len(waits) == 3


# ---------------------------------------------------------------------------
# C entries: refused before anything is launched (the addresses are never read)
# ---------------------------------------------------------------------------
ERR_ARG = -1
ADDR = ctypes.c_void_p(4096)


class Side(ctypes.Structure):
    _fields_ = [("n_rows", ctypes.c_int64), ("n_cols", ctypes.c_int64),
                ("n_edges", ctypes.c_int64), ("plan", ctypes.c_void_p),
                ("n_items", ctypes.c_int32), ("n_parts", ctypes.c_int32)]


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(os.path.join(REPO, "batmobile-evo_amd", "lib", "libbatmobile_hip.so"))


def _attention(lib, side, **given):
    """batteries_neighbor_attention with 2 heads of 16, f32."""
    p = {**dict.fromkeys(("q", "k", "v", "out"), ADDR), **given}
    i64, none = ctypes.c_int64, ctypes.c_void_p(None)
    return lib.batteries_neighbor_attention(
        p["q"], p["k"], p["v"], none, none, 0, ctypes.byref(side), p["out"], none, 2, 2, 16, 16,
        i64(32), i64(32), i64(32), ctypes.c_float(1.0), 0, none, ctypes.c_size_t(0), none)


@pytest.mark.parametrize("n_edges,missing", [(0, "q"), (0, "out"), (5, "q"), (5, "k"), (5, "v"),
                                             (5, "out")])
def test_attention_refuses_a_missing_array(lib, n_edges, missing):
    """q and out are read and written for every row, also where no row has an edge; k and v only
    along edges."""
    side = Side(3, 4, n_edges, 4096, 1, 0)
    assert _attention(lib, side, **{missing: None}) == ERR_ARG


# ---------------------------------------------------------------------------
# forward-mode derivatives: refused before anything else, never dropped
# ---------------------------------------------------------------------------

def _attention_call(batmobile, q, k, v, bias):
    plan = types.SimpleNamespace(n_dst=3, n_src=4, side=(torch.zeros(0, dtype=torch.int32), 0, 0),
                                 src=torch.zeros(2), edge_id=None, row_ptr=torch.zeros(4),
                                 source_side=lambda: None)
    return batmobile.neighbor_attention(q, k, v, plan, bias=bias)


TANGENT_CALLS = {
    "neighbor_attention": (_attention_call, [(3, 2, 8), (4, 2, 8), (4, 2, 8), (2, 2)]),
    "equivariant_norm": (lambda b, x, w: b.equivariant_norm(x, w), [(3, 5, 16), (4, 5)]),
    "gated_residual_norm": (lambda b, *t: b.gated_residual_norm(*t),
                            [(3, 5, 16), (3, 5, 16), (3, 5, 4), (5,), (4, 5), (4, 5)]),
    "clip_grad_norm": (lambda b, *t: b.clip_grad_norm(list(t), 1.0), [(3,), (4, 5)]),
}


@pytest.mark.parametrize("name,at", [(n, i) for n, (_, s) in TANGENT_CALLS.items()
                                     for i in range(len(s))])
@pytest.mark.parametrize("others_need_grad", [False, True])
def test_forward_mode_derivatives_are_refused(name, at, others_need_grad):
    import batmobile
    import torch.autograd.forward_ad as fw
    call, shapes = TANGENT_CALLS[name]
    args = [torch.ones(s, requires_grad=others_need_grad and i != at) for i, s in enumerate(shapes)]
    with fw.dual_level():
        args[at] = fw.make_dual(torch.ones(shapes[at]), torch.ones(shapes[at]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(batmobile, *args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(batmobile, *args)
    with pytest.raises(RuntimeError, match="CUDA"):      # without a tangent: the next check
        call(batmobile, *[torch.ones(s) for s in shapes])
