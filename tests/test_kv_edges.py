"""The paged cache's calls at the ends of what they take, on the CPU: empty page tables, pools without a pitch, numbers past 32 bits."""
from __future__ import annotations

import pytest
import torch

import ascq
from test_block_checks import _refused
from test_block_launches import _run


def test_workspace_sizes_of_an_empty_page_table():
    """a table narrowed to the pages of sequences that are all empty has no columns, and no memory; the calls take it"""
    cache = ascq.kv_cache(4, 2, 16, 128, 32, device="cpu")
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    table = torch.zeros(3, 2, dtype=torch.int32)
    for none in (table[:, :0], torch.zeros(3, 0, dtype=torch.int32)):
        assert ascq.kv_attention_workspace_size(q, cache, none) == 0
        assert ascq.kv_attention_workspace_size(q, cache, none, starts=torch.zeros(4, dtype=torch.int32), max_queries=2) == 0
        assert ascq.kv_evict_workspace_size(cache, none) == 0
    assert ascq.kv_attention_workspace_size(q[:0], cache, table[:0]) == 0
    assert ascq.kv_evict_workspace_size(cache, table[:0]) == 0


def test_pools_without_a_pitch_are_refused():
    """pages that all lie in one place (a page expanded to several): the library takes a pitch of 0 as that of dense pools"""
    one, good = (ascq.kv_cache(n, 2, 16, 128, 32, device="cpu") for n in (1, 8))
    parts = list(good)
    for i, t in enumerate(one):
        _refused(ascq.KvCache, *[t.expand(8, *t.shape[1:]) if i == j else x for j, x in enumerate(parts)])
    _refused(ascq.KvCache, *[t.expand(8, *t.shape[1:]) for t in one])
    ascq.KvCache(*one)
    ascq.KvCache(*[t.expand(1, *t.shape[1:]) for t in one])


def test_evict_numbers_past_32_bits():
    """what the library's 32-bit fields cannot hold is refused, not cut to its low bits"""
    cache = ascq.kv_cache(4, 2, 16, 128, 32, device="cpu")
    table, n, w = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, 32)
    for keep, recent in ((8, (1 << 32) + 1), (8, 1 << 32), (8, -(1 << 32)), (8, 9), (8, -1), ((1 << 32) + 8, 0)):
        with pytest.raises(ascq.AscqError, match="keep"):
            ascq.kv_evict(cache, table, n, w, keep, recent)


def test_weights_on_the_cpu_are_refused():
    """before anything is copied or a stream is asked for"""
    cache = ascq.kv_cache(4, 2, 16, 128, 32, device="cpu")
    q, lse, w = torch.zeros(3, 4, 128).half(), torch.zeros(3, 4), torch.zeros(3, 2, 32)
    table, n = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for kw in (dict(), dict(stream=5), dict(out=w)):
        _refused(ascq.kv_weights, q, lse, cache, table, n, weights=w, **kw)


def test_evict_of_the_longest_tables(tmp_path):
    """tables of up to 2^30 tokens over up to 1024 key heads: no grid of 2^32 threads"""
    _run(tmp_path, "kv_wide")
