"""Attention, norms and clipping without a GPU: what is refused on the host before anything runs,
and the order of work around a plan's wait."""
import types

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


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
