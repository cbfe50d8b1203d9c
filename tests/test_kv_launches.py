"""The paged cache's launches (CPU only): the built library driven by a program that records them."""
from __future__ import annotations

from test_block_launches import _run


def test_launches_cover_every_call(tmp_path):
    """very many tokens, sequences, queries and pages: everything once, no grid past its limits, no write past the workspace"""
    _run(tmp_path, "kv_launches")
