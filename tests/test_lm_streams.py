"""Streams that the language-model operators of the ctypes harness are given (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from hfuse_b200 import ops


def test_a_stream_of_another_device_is_refused():
    """kernels launched there would be handed this device's addresses"""
    x = SimpleNamespace(device=torch.device("cuda", 0))
    here, there = (SimpleNamespace(device=torch.device("cuda", k), cuda_stream=0) for k in (0, 1))
    assert ops._on(x, here).stream is here
    with pytest.raises(ValueError, match="stream"):
        ops._on(x, there)
