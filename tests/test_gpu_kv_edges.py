"""The paged cache where a call's masks, tiles and turns end inside its steps: rows that no query sees hold anything, and many
queries' weights are added up in several turns over the tokens."""
from __future__ import annotations

import math

import pytest
import torch

import kv_lib as K
from test_gpu_kv import _check_attention

pytestmark = pytest.mark.gpu

SHAPES = [(64, 32), (64, 64), (128, 32), (128, 128), (256, 32), (256, 128)]
# queries of each sequence (None: one each), lengths, heads (two key heads), window: a step begins up to 31 tokens before the first
# that any row sees, a whole page and more of them.  One query: (2000, 984) begins at token 1016, its step at 992.  5 x 4 rows are two
# tiles of 16; 60, 80 and 400 rows share converted steps, in tiles of 64 to 256 rows.
WINDOWS = [(None, [2000, 70, 333, 1001, 17, 0], 8, 984), (None, [2000, 70, 333, 1001, 17, 0], 8, 21), (None, [5000], 4, 4500),
           ([5, 1, 4], [99, 200, 1000], 8, 33), ([15, 2], [333, 40], 8, 50), ([40, 3, 0, 17], [333, 64, 20, 19], 4, 37), ([100, 70], [1000, 160], 8, 45)]


def _unseen(p, causal, window):
    """tokens [batch, table's tokens] that no query of their sequence sees"""
    t = torch.arange(p.columns * p.page)
    out = torch.ones(len(p.lengths), t.numel(), dtype=torch.bool)
    for b, length in enumerate(p.lengths):
        for i in range(p.queries[b]):
            at = length - p.queries[b] + i
            out[b] &= ~((t < length) & (t > at - window) & ((t <= at) | (not causal)))
    return out


def _spoil(p, unseen, which, given_back):
    """every (scale, offset) pair of such tokens becomes NaN, infinite or large, as are those of the spare pages; given_back: whole
    pages of them are no longer the sequence's, their columns name a spare page"""
    bad = torch.tensor([math.nan, math.inf, -math.inf, 65504.0]).half()
    for w in which:
        pool = p.cache[w]
        fill = bad[torch.randint(0, 4, pool.shape, generator=p.g)]
        spoiled = torch.zeros(pool.shape[0], p.page, dtype=torch.bool)
        spoiled[p.spare.long()] = True
        for b in range(len(p.lengths)):
            for t in unseen[b].nonzero().flatten().tolist():
                page = int(p.table[b, t // p.page])
                if page >= 0:
                    spoiled[page, t % p.page] = True
        p.cache[w] = torch.where(spoiled[:, None, :, None, None], fill, pool)
    if given_back:
        whole = unseen.view(len(p.lengths), p.columns, p.page).all(dim=2)
        p.table = torch.where(whole & (p.table >= 0), p.spare[0], p.table)


@pytest.mark.parametrize("given_back", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,group", SHAPES)
def test_attention_garbage_before_the_window(ascq_gpu, d, group, causal, given_back):
    """nothing of a token that no query sees reaches a result: equal bits with and without the garbage"""
    for i, (queries, lengths, heads, window) in enumerate(WINDOWS):
        p = K.Problem(d + i, lengths, queries=queries, heads=heads, kv=2, d=d, group=group, page=16, dt="bf16" if i % 2 else "f16")
        want = _check_attention(ascq_gpu, p, causal=causal, window=window)
        _spoil(p, _unseen(p, causal, window), (2, 3), given_back)
        args, more = p.args(ascq_gpu)
        got = ascq_gpu.kv_attention(*args, **more, need_lse=True, causal=causal, window=window)
        for a, b in zip(got, want):
            assert torch.isfinite(a[torch.isfinite(b)]).all(), (queries, window)
            assert torch.equal(a, b), (queries, window)


@pytest.mark.parametrize("given_back", [False, True])
@pytest.mark.parametrize("d,group", SHAPES)
def test_weights_garbage_before_the_window(ascq_gpu, d, group, given_back):
    """weights of tokens that no query sees are decay times what they were, whatever those tokens' keys are"""
    for i, (queries, lengths, heads, window) in enumerate(WINDOWS):
        p = K.Problem(d + i, lengths, queries=queries, heads=heads, kv=2, d=d, group=group, page=16, dt="bf16" if i % 2 else "f16")
        args, more = p.args(ascq_gpu)
        _, lse = ascq_gpu.kv_attention(*args, **more, need_lse=True, window=window)
        unseen = _unseen(p, True, window)
        cap = unseen.shape[1]
        before = torch.rand(len(lengths), p.kv, cap, generator=p.g)
        want = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, weights=before.cuda(), decay=0.5, window=window)
        _spoil(p, unseen, (2,), given_back)
        args, more = p.args(ascq_gpu)
        got = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, weights=before.cuda(), decay=0.5, window=window)
        fresh = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, window=window)
        inside = torch.arange(cap)[None, :] < torch.tensor(lengths)[:, None]
        for h in range(p.kv):
            kept = got[:, h].cpu()
            assert torch.equal(kept[unseen & inside], 0.5 * before[:, h][unseen & inside]), (queries, window)
            assert torch.equal(kept[unseen & ~inside], before[:, h][unseen & ~inside]), (queries, window)
            assert torch.all(fresh[:, h].cpu()[unseen] == 0), (queries, window)
        assert torch.equal(got, want), (queries, window)


@pytest.mark.parametrize("queries,window", [(70, 0), (150, 0), (150, 2500)])
@pytest.mark.parametrize("d,group,dt", [(64, 64, "f16"), (128, 32, "bf16"), (256, 64, "f16")])
def test_weights_in_turns(ascq_gpu, d, group, dt, queries, window):
    """280 and 600 rows: two or three turns of 256 (d 256: three or five of 128) over ranges of several steps a wave, each adding to what
    the turn before left.  64 sequences, of which one is long, give ranges of 1536 tokens (d 256: 1280): three steps of the eight
    waves and more."""
    p = K.Problem(queries + d, [4401] + [3] * 63, queries=[queries, 1] + [0] * 62, heads=4, kv=1, d=d, group=group, page=64, dt=dt)
    args, more = p.args(ascq_gpu)
    kw = dict(window=window)
    _, lse = ascq_gpu.kv_attention(*args, **more, need_lse=True, **kw)
    *_, want, tol = K.attention(p, **kw)
    cap = p.columns * p.page
    before = torch.rand(64, 1, cap, generator=p.g)
    fresh = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, out=torch.full(before.shape, math.nan).cuda(), **kw).cpu()
    place = before.cuda()
    for _ in range(3):  # (the same bits from the same inputs)
        place.copy_(before)
        ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, weights=place, decay=0.5, out=place, **kw)
        apart = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, weights=before.cuda(), decay=0.5, **kw)
        assert torch.equal(apart, place)
    for b, n in enumerate(p.lengths):
        w, e = want[b][:, :n], tol[b][:, :n]
        assert torch.all((fresh[b, :, :n].double() - w).abs() <= e + 2.0 ** -24)
        assert torch.all(fresh[b, :, n:] == 0)
        total = 0.5 * before[b, :, :n].double() + w
        assert torch.all((place[b, :, :n].cpu().double() - total).abs() <= e + 2.0 ** -23 * total + 2.0 ** -24)
        assert torch.equal(place[b, :, n:].cpu(), before[b, :, n:])


def test_an_empty_page_table(ascq_gpu):
    """sequences that are all empty, the table narrowed to no column: zeros and -inf, zero weights, nothing kept"""
    a, cache = ascq_gpu, ascq_gpu.kv_cache(4, 2, 16, 128, 32)
    table, n = torch.zeros(3, 2, dtype=torch.int32, device="cuda")[:, :0], torch.zeros(3, dtype=torch.int32, device="cuda")
    for starts, most in (([0, 1, 2, 3], 1), ([0, 4, 5, 60], 55)):
        q = torch.randn(starts[-1], 4, 128, device="cuda").half()
        kw = {} if most == 1 else dict(starts=torch.tensor(starts).int().cuda(), max_queries=most)
        out, lse = a.kv_attention(q, cache, table, n, need_lse=True, **kw,
                                  workspace=torch.empty(a.kv_attention_workspace_size(q, cache, table, **kw), dtype=torch.uint8, device="cuda"))
        assert torch.all(out == 0) and torch.all(lse == -math.inf)
        w = a.kv_weights(q, lse, cache, table, n, out=torch.full((3, 2, 7), math.nan, device="cuda"), **kw)
        assert torch.all(w == 0)
    room = torch.empty(a.kv_evict_workspace_size(cache, table), dtype=torch.uint8, device="cuda")
    kept, m, w = a.kv_evict(cache, table, n, torch.ones(3, 2, 7, device="cuda"), 5, 2, workspace=room)
    assert torch.all(kept == -1) and torch.all(m == 0) and torch.all(w == 0)
