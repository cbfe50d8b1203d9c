"""The block operators' host side at the edges of their ranges (CPU only): what a call refuses, plans and launches."""
from __future__ import annotations

import ctypes

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


def _linear_room(m, n, k, ld_w=0, trans=1):
    p = ascq._LinearParam(m, n, k, 0, ld_w, 0, 0, ascq.INT8, ascq.F16, trans, 0)
    need = ctypes.c_size_t(0)
    assert ascq.lib().ascq_quant_linear_workspace_size(0x10000, 0x20000, ctypes.byref(p), ctypes.byref(need)) == ascq.OK
    return need.value


@pytest.mark.parametrize("m,n,k,rows", [(40, 4096, 65536, True), (200, 4096, 65536, True), (200, 128, 65536, False),
                                        (70, 200, 65536, False)])
def test_workspace_of_the_last_piece(m, n, k, rows):
    """operands past 2^31 bytes go in pieces; a short last one shares its K among workgroups, whose sums need their room"""
    piece = ((1 << 31) - 16) // k // 256 * 256
    alone = _linear_room(m, n, k)
    assert alone > 0
    whole = _linear_room(piece, n, k) if rows else _linear_room(m, piece, k)
    got = _linear_room(2 * piece + m, n, k) if rows else _linear_room(m, 2 * piece + n, k)
    assert got == max(alone, whole)
    assert (_linear_room(2 * piece, n, k) if rows else _linear_room(m, 2 * piece, k)) == whole
