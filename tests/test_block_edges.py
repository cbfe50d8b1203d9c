"""The block operators' host side at the edges of their ranges (CPU only): what a call refuses, plans and launches."""
from __future__ import annotations

import pytest
import torch

import ascq


def test_workspace_must_be_one_run():
    """a view with gaps, or one that repeats an element, has fewer bytes behind its first than it has elements: refused"""
    x, w = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(32, 64, dtype=torch.int8)
    logits = torch.zeros(100, 8)
    strided = torch.zeros(4096, dtype=torch.uint8)[::2]
    repeated = torch.zeros(1, dtype=torch.uint8).expand(1 << 20)
    for ws in (strided, repeated):
        with pytest.raises(ascq.AscqError, match="workspace must be contiguous") as e:
            ascq.quant_linear(x, torch.ones(4), w, torch.ones(32), workspace=ws)
        assert e.value.status == ascq.E_INVALID_ARG
        with pytest.raises(ascq.AscqError, match="workspace must be contiguous") as e:
            ascq.moe_route(logits, 2, workspace=ws)
        assert e.value.status == ascq.E_INVALID_ARG
