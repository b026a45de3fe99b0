"""Tests that need no GPU run where none can be reached."""
import os


def test_no_gpu_is_visible():
    """C entries are handed addresses that lead nowhere and refuse the call; were a refusal lost, the launch
    has to end as an error code."""
    import torch
    assert os.environ["HIP_VISIBLE_DEVICES"] == "-1"
    assert not torch.cuda.is_available()
