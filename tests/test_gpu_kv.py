"""Attention over the paged int4 cache (ascq_kv_*) against plain 64-bit implementations (tests/kv_lib.py, where the bounds are
derived).  Codes, scales, offsets, positions, lengths and moved rows are equal bit for bit."""
from __future__ import annotations

import math

import pytest
import torch

import kv_lib as K

pytestmark = pytest.mark.gpu


def _check_attention(ascq, p, got=None, **kw):
    args, more = p.args(ascq)
    out, lse = got or ascq.kv_attention(*args, **more, need_lse=True, **kw)
    want, want_lse, tol, tol_lse, *_ = K.attention(p, **kw)
    o, l = out.double().cpu(), lse.double().cpu()
    half = K.HALF[p.dt]
    assert torch.all((o - want).abs() <= tol * (1 + half) + half * want.abs() + 2.0 ** -25)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(l) & (l < 0), empty)
    assert torch.all(o[empty] == 0)
    assert torch.all((l - want_lse).abs()[~empty] <= tol_lse[~empty])
    return out, lse


# ---------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_append(ascq_gpu, d, group, dt):
    kv, page, t = 3, 32, 41
    g = torch.Generator().manual_seed(d + group)
    k, v = (torch.randn(t, kv, d, generator=g).to(K.DT[dt]) for _ in range(2))
    k[0] = 0.0                      # a group without a range
    k[1] = 1.5
    k[2, :, 3] = math.nan           # counts as 0
    k[3, :, 5], k[4, :, 6] = math.inf, -math.inf
    k[5] = torch.finfo(K.DT[dt]).max
    k[6, :, ::2], k[6, :, 1::2] = 61440.0, -61440.0
    k[7] = k[7] * 1e-7              # scales below f16's normal numbers
    k[8] = k[8] * 1e-9
    k[9] = k[9] + 100               # a large offset
    v[0, :, 1::3] = -0.0
    pages = 5
    slots = torch.randperm(pages * page, generator=g)[:t]
    slots[10], slots[11], slots[12] = -1, pages * page, -(1 << 40)
    cache = ascq_gpu.KvCache(*(torch.full(s, 0x5A, dtype=torch.uint8).cuda() for s in [(pages, kv, page, d // 2)] * 2),
                             *(torch.full((pages, kv, page, d // group, 2), 7.0).half().cuda() for _ in range(2)))
    before = [x.clone() for x in cache]
    ascq_gpu.kv_append(cache, k.cuda(), v.cuda(), slots.cuda())
    want = [x.cpu().clone() for x in before]
    for x, codes, scales in ((k, want[0], want[2]), (v, want[1], want[3])):
        c, s, o = K.quantize(x, group)
        packed, pairs = K.pack(c), torch.stack([s, o], dim=-1)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                codes[slot // page, :, slot % page] = packed[i]
                scales[slot // page, :, slot % page] = pairs[i]
    for a, b in zip(cache, want):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    assert all(torch.isfinite(K.values(a.cpu(), b.cpu())).all() for a, b in zip(list(cache)[:2], list(cache)[2:]))


@pytest.mark.parametrize("d,group", [(64, 64), (128, 32), (256, 128)])
def test_append_error(ascq_gpu, d, group):
    """a value is within half a step of what was appended, a step being the group's range / 15, and the roundings of scale and
    offset: 2^-11 (15 step + |offset|), and the value's own"""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 2, d, generator=g).half()
    cache = ascq_gpu.kv_cache(4, 2, 16, d, group)
    ascq_gpu.kv_append(cache, x.cuda(), (2 * x).cuda(), torch.arange(64).cuda())
    for which, want in ((0, x), (1, 2 * x)):
        got = K.values(list(cache)[which].cpu(), list(cache)[which + 2].cpu()).transpose(1, 2).flatten(0, 1)
        r = want.double().unflatten(-1, (-1, group))
        step = ((r.amax(-1) - r.amin(-1)) / 15).repeat_interleave(group, dim=-1)
        big = r.abs().amax(-1).repeat_interleave(group, dim=-1)
        assert torch.all((got - want.double()).abs() <= 0.5 * step + 2.0 ** -11 * (15 * step + 3 * big))


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_append_strides(ascq_gpu, dt):
    """slices of a fused projection, heads before tokens, rows off 16 bytes, pools with gaps between pages"""
    kv, d, group, t = 2, 128, 64, 20
    g = torch.Generator().manual_seed(4)
    fused = torch.randn(t, 4 + 2 * kv, d, generator=g).to(K.DT[dt]).cuda()
    slots = torch.randperm(32, generator=g)[:t].cuda()
    plain = ascq_gpu.kv_cache(2, kv, 16, d, group)
    for x in plain:
        x.zero_()
    ascq_gpu.kv_append(plain, fused[:, 4:6].contiguous(), fused[:, 6:].contiguous(), slots)
    both = torch.zeros(2, 2, kv, 16, d // 2, dtype=torch.uint8, device="cuda")
    pairs = torch.zeros(2, 2, kv, 16, d // group, 2, dtype=torch.float16, device="cuda")
    odd = torch.empty(t * kv * (d + 3) + 1, dtype=K.DT[dt], device="cuda")[1:].view(t, kv, d + 3)[:, :, :d]
    odd.copy_(fused[:, 6:])
    for k, v in ((fused[:, 4:6], fused[:, 6:]), (fused[:, 4:6].transpose(0, 1).contiguous().transpose(0, 1), odd)):
        both.zero_()
        pairs.zero_()
        cache = ascq_gpu.KvCache(both[:, 0], both[:, 1], pairs[:, 0], pairs[:, 1])
        ascq_gpu.kv_append(cache, k, v, slots)
        assert all(torch.equal(a, b) for a, b in zip(cache, plain))


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_attention_one_query(ascq_gpu, d, group, dt):
    for page, heads, kv in ((16, 4, 2), (32, 7, 1), (64, 3, 3), (128, 40, 2)):
        p = K.Problem(d + group + page, [1, 15, 16, 17, 31, 32, 33, 100, 129, 300], heads=heads, kv=kv, d=d, group=group, page=page,
                      dt=dt, q_size=1.5)
        _check_attention(ascq_gpu, p)


@pytest.mark.parametrize("length", [1, 2, 127, 128, 129, 255, 256, 257, 1000, 4099, 20011])
def test_attention_lengths(ascq_gpu, length):
    p = K.Problem(length, [length], heads=4, kv=2, page=32, group=64)
    _check_attention(ascq_gpu, p)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 32), (256, 64)])
def test_attention_queries(ascq_gpu, d, group, causal):
    """several queries a sequence, more of them than tokens, none of them; tiles that end inside a query's heads"""
    p = K.Problem(9, [5, 40, 3, 0, 77, 130, 64, 12], queries=[5, 7, 8, 2, 0, 50, 33, 1], heads=6, kv=2, d=d, group=group, page=16,
                  dt="bf16")
    _check_attention(ascq_gpu, p, causal=causal)
    _check_attention(ascq_gpu, p, causal=causal, window=9)


@pytest.mark.parametrize("ratio,kv", [(1, 2), (4, 1), (7, 1)])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_attention_many_queries(ascq_gpu, d, group, ratio, kv):
    """tiles of 64 to 256 rows, in part filled; sequences of fewer tokens than queries; more rows than one tile"""
    for queries, lengths, page, dt in (([40], [70], 16, "f16"), ([100, 3], [100, 9], 32, "bf16"), ([70, 1, 200], [300, 33, 150], 64, "f16")):
        p = K.Problem(d + ratio, lengths, queries=queries, heads=ratio * kv, kv=kv, d=d, group=group, page=page, dt=dt)
        _check_attention(ascq_gpu, p)
        _check_attention(ascq_gpu, p, window=37)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 1 << 40])
def test_attention_window(ascq_gpu, window):
    p = K.Problem(window % 1000, [1, 31, 64, 99, 333], heads=4, kv=4, page=16, d=64, group=64)
    _check_attention(ascq_gpu, p, window=window)
    p = K.Problem(3, [60, 20, 200], queries=[20, 20, 65], heads=4, kv=2, page=32)
    _check_attention(ascq_gpu, p, window=window)


def test_attention_scale(ascq_gpu):
    p = K.Problem(5, [200, 64], heads=4, kv=2, page=16)
    for scale in (1.0, 0.0, -0.25, 1e-6):
        _check_attention(ascq_gpu, p, scale=scale)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_sizes_of_queries(ascq_gpu, dt):
    """rows of very small and very large queries, and of zeros: every row is scaled by itself"""
    p = K.Problem(6, [150, 150], heads=8, kv=1, page=16, dt=dt)
    size = torch.tensor([1.0, 0.0, 1e-4, 3e-7, 30.0, 1e-2, 5.0, 2.0 ** -24])
    p.q = (p.q.double() * size[None, :, None]).to(p.q.dtype)
    _check_attention(ascq_gpu, p)
    if dt == "bf16":
        p.q = (torch.randn(p.q.shape, generator=p.g).double() * torch.tensor([1e-38, 1e-30, 1e-20, 1e-10, 1, 10, 50, 1e-39])[None, :, None]).to(p.q.dtype)
        _check_attention(ascq_gpu, p)


@pytest.mark.parametrize("kv_size", [1e-6, 1e-4, 100.0, 15000.0])
def test_attention_sizes_of_values(ascq_gpu, kv_size):
    """values down to f16's subnormals and up to its end"""
    p = K.Problem(7, [100, 37], heads=4, kv=2, page=16, kv_size=kv_size)
    _check_attention(ascq_gpu, p, scale=0.1 / kv_size)


def test_attention_sharp_and_late_maximum(ascq_gpu):
    """scores that rise by hundreds along the sequence, so that the running maximum moves often, and fall"""
    p = K.Problem(8, [600, 600], heads=4, kv=1, page=16, d=64)
    k = torch.randn(p.cache[0].shape[0], 1, 16, 64, generator=p.g)
    for b in range(2):
        for t in range(600):
            k[p.table[b, t // 16], 0, t % 16, 0] = (t if b == 0 else 600 - t) / 20.0
    c, s, o = K.quantize(k, 32)
    p.cache[0], p.cache[2] = K.pack(c), torch.stack([s, o], dim=-1)
    p.q[:, :, 0] = torch.tensor([1.0, 20.0, 60.0, -60.0]).half()
    _check_attention(ascq_gpu, p)


def test_attention_garbage_behind_the_end(ascq_gpu):
    """NaN and infinite scales behind a sequence's length, on pages of nobody, and in queries of other rows"""
    p = K.Problem(10, [5, 33, 0, 47, 160], queries=[2, 1, 1, 3, 9], heads=4, kv=2, page=16)
    want = K.attention(p)
    bad = torch.tensor([math.nan, math.inf, -math.inf, 65504.0]).half()
    for which in (2, 3):
        pool = p.cache[which]
        live = torch.zeros(pool.shape[0], 16, dtype=torch.bool)
        for b, n in enumerate(p.lengths):
            for t in range(n):
                live[p.table[b, t // 16], t % 16] = True
        fill = bad[torch.randint(0, 4, pool.shape, generator=p.g)]
        p.cache[which] = torch.where(live[:, None, :, None, None], pool, fill)
    args, more = p.args(ascq_gpu)
    out, lse = ascq_gpu.kv_attention(*args, **more, need_lse=True)
    assert torch.all((out.cpu().double() - want[0]).abs() <= want[2] * 1.001 + 2.0 ** -11 * want[0].abs() + 2.0 ** -25)
    p.q[0], p.q[5, 1] = math.nan, math.inf
    args, more = p.args(ascq_gpu)
    bad_out, _ = ascq_gpu.kv_attention(*args, **more)
    assert torch.isnan(bad_out[0]).all() and torch.isnan(bad_out[5, 1]).all()
    same = torch.ones(out.shape[:2], dtype=torch.bool)
    same[0], same[5, 1] = False, False
    assert torch.equal(bad_out.cpu()[same], out.cpu()[same])


def test_attention_bad_tables(ascq_gpu):
    """pages outside the cache mask their tokens, lengths end at the table, starts outside q give nothing"""
    p = K.Problem(11, [100, 80, 64, 50], heads=4, kv=2, page=16)
    pages = p.cache[0].shape[0]
    p.table[0, 2], p.table[0, 4], p.table[1, 0], p.table[2, :] = -5, pages, 1 << 30, -1
    p.lengths = [100, 1 << 30, 64, -7]
    _check_attention(ascq_gpu, p)
    p = K.Problem(12, [40, 30, 20], queries=[2, 3, 1], heads=4, kv=2, page=16)
    args, more = p.args(ascq_gpu)
    good, _ = ascq_gpu.kv_attention(*args, **more)
    for starts in ([0, 2, 5, 1 << 20], [0, 2, 5, -3], [-4, 2, 5, 6]):
        out = torch.full_like(good, 77.0)
        more["starts"] = torch.tensor(starts).int().cuda()
        ascq_gpu.kv_attention(*args, **more, out=out)
        for b in range(3):
            rows = slice(int(p.starts[b]), int(p.starts[b + 1]))
            if starts[b:b + 2] == p.starts[b:b + 2].tolist():
                assert torch.equal(out[rows], good[rows])


def test_attention_strides_and_rows_of_nobody(ascq_gpu):
    """queries and outputs of any pitch and alignment; rows behind the last sequence stay as they were; narrowed page tables"""
    p = K.Problem(13, [50, 20, 90], queries=[3, 1, 4], heads=4, kv=2, page=16, columns=9)
    args, more = p.args(ascq_gpu)
    want, want_lse = ascq_gpu.kv_attention(*args, **more, need_lse=True)
    t, h, d = want.shape
    wide = torch.zeros(t + 2, h + 3, d, dtype=torch.float16, device="cuda")
    wide[:t, 1:h + 1] = args[0]
    out = torch.full((t + 2, h, d), 3.0, dtype=torch.float16, device="cuda")
    lse = torch.full((t + 2, h), 3.0, device="cuda")
    ascq_gpu.kv_attention(wide[:, 1:h + 1], *args[1:], **more, out=out, lse=lse)
    assert torch.equal(out[:t], want) and torch.equal(lse[:t], want_lse)
    assert torch.all(out[t:] == 3) and torch.all(lse[t:] == 3)
    odd = torch.zeros(h * t * (d + 1) + 1, dtype=torch.float16, device="cuda")
    q = odd[1:].view(h, t, d + 1)[:, :, :d].transpose(0, 1)  # heads first, rows off every alignment
    q.copy_(args[0])
    res = torch.zeros_like(odd)[1:].view(h, t, d + 1)[:, :, :d].transpose(0, 1)
    ascq_gpu.kv_attention(q, *args[1:], **more, out=res)
    assert torch.equal(res, want)
    ascq_gpu.kv_attention(q, args[1], args[2][:, :6], args[3], **more, out=res)
    assert torch.equal(res, want)
    both = torch.stack(list(args[1])[:2], dim=1).contiguous()
    pairs = torch.stack(list(args[1])[2:], dim=1).contiguous()
    ascq_gpu.kv_attention(q, ascq_gpu.KvCache(both[:, 0], both[:, 1], pairs[:, 0], pairs[:, 1]), *args[2:], **more, out=res)
    assert torch.equal(res, want)


def test_attention_workspace(ascq_gpu):
    """with its workspace, with less, without: within the bounds each; the same bits every time"""
    p = K.Problem(14, [5000, 3000], heads=4, kv=1, page=64, group=128)
    args, more = p.args(ascq_gpu)
    need = ascq_gpu.kv_attention_workspace_size(args[0], args[1], args[2])
    assert need > 0
    want = K.attention(p)
    for size in (need, need - 1, 0):
        room = torch.full((size + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        got = ascq_gpu.kv_attention(*args, need_lse=True, workspace=room[:size])
        assert torch.all((got[0].cpu().double() - want[0]).abs() <= want[2] * 1.001 + 2.0 ** -11 * want[0].abs() + 2.0 ** -25)
        assert torch.all((got[1].cpu().double() - want[1]).abs() <= want[3])
        assert torch.all(room[size:] == 0xFF)
        for _ in range(3):
            again = ascq_gpu.kv_attention(*args, need_lse=True, workspace=room[:size])
            assert all(torch.equal(a, b) for a, b in zip(got, again))


# ---------------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("d,group,dt", [(64, 32, "f16"), (64, 64, "bf16"), (128, 32, "bf16"), (128, 64, "f16"), (128, 128, "bf16"),
                                        (256, 32, "f16"), (256, 64, "bf16"), (256, 128, "f16")])
def test_weights(ascq_gpu, d, group, dt):
    for kw in (dict(), dict(window=21), dict(causal=False)):
        p = K.Problem(d, [1, 40, 3, 0, 200, 130], queries=[1, 7, 5, 2, 0, 50], heads=6, kv=2, d=d, group=group, page=16, dt=dt)
        args, more = p.args(ascq_gpu)
        _, lse = ascq_gpu.kv_attention(*args, **more, need_lse=True, **kw)
        *_, want, tol = K.attention(p, **kw)
        cap = p.columns * p.page + 5
        before = torch.rand(len(p.lengths), p.kv, cap, generator=p.g)
        fresh = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more, out=torch.full(before.shape, math.nan).cuda(), **kw).cpu()
        place = before.cuda()
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


def test_weights_add_up(ascq_gpu):
    """each query of a head gives 1 in all"""
    p = K.Problem(3, [3000, 700], queries=[40, 3], heads=8, kv=2, page=32)
    args, more = p.args(ascq_gpu)
    _, lse = ascq_gpu.kv_attention(*args, **more, need_lse=True)
    w = ascq_gpu.kv_weights(args[0], lse, *args[1:], **more)
    want = torch.tensor(p.queries, dtype=torch.float64)[:, None].expand(2, 2) * 4
    assert torch.all((w.double().sum(dim=2).cpu() - want).abs() <= 1e-4 * want)


# ---------------------------------------------------------------------------------------------- evict
def _check_evict(ascq, p, w, keep, recent, into=None, cap_out=None, **more):
    cache = p.gpu(ascq)
    before = [x.cpu().clone() for x in cache]
    wt = w.cuda()
    out = None if cap_out is None else torch.full((*w.shape[:2], cap_out), math.nan).cuda()
    n0 = torch.tensor(p.lengths).int().cuda()
    kept, n, got = ascq.kv_evict(cache, p.table.cuda(), n0, wt, keep, recent, into=None if into is None else into.cuda(),
                                 weights_out=out, **more)
    assert n.tolist() == [min(x, keep) for x in p.lengths]
    want = [x.clone() for x in before]
    for b, length in enumerate(p.lengths):
        for h in range(p.kv):
            stay = K.evict(w[b, h], length, keep, recent)
            assert kept[b, h].tolist() == stay + [-1] * (keep - len(stay))
            row = torch.zeros(got.shape[2])
            row[:len(stay)] = w[b, h][stay]
            assert torch.equal(got[b, h].cpu().nan_to_num(nan=-5.0), row.nan_to_num(nan=-5.0))
            i, t = torch.arange(len(stay)), torch.tensor(stay, dtype=torch.long)
            src = p.table[b].long()[t // p.page]
            dst = (p.table if into is None else into)[b].long()[i // p.page]
            for pool, old in zip(want, before):
                pool[dst, h, i % p.page] = old[src, h, t % p.page]
    for a, b in zip(cache, want):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    if out is not None:
        assert torch.equal(wt.cpu().nan_to_num(nan=-5.0), w.nan_to_num(nan=-5.0))


@pytest.mark.parametrize("away", [False, True])
@pytest.mark.parametrize("d,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)])
def test_evict(ascq_gpu, d, group, away):
    lengths, page = [1, 30, 64, 65, 100, 257, 0, 40], 16
    for keep, recent in ((40, 8), (64, 0), (33, 33), (1, 1), (1, 0)):
        p = K.Problem(keep, lengths, heads=2, kv=2, d=d, group=group, page=page, spare=40)
        cap = p.columns * page
        w = torch.rand(len(lengths), 2, cap, generator=p.g)
        w = torch.where(torch.rand(w.shape, generator=p.g) < 0.5, (w * 4).round() / 4, w)  # equal ones, zeros
        w[0, 0, 0], w[4, 1, 3], w[5, 0, 7], w[5, 1, 11] = math.nan, math.nan, -0.0, -1.0
        into = p.spare[:len(lengths) * 5].view(len(lengths), 5) if away else None
        _check_evict(ascq_gpu, p, w, keep, recent, into, cap_out=keep + 7 if away else None)


@pytest.mark.parametrize("alone", [False, True])
@pytest.mark.parametrize("away", [False, True])
@pytest.mark.parametrize("keep,recent", [(9500, 1000), (1, 0), (5000, 5000), (8193, 1), (14000, 30)])
def test_evict_long(ascq_gpu, keep, recent, away, alone):
    """tens of thousands of tokens, in place and elsewhere, with and without the workspace; all weights equal, all zero but few,
    weights that differ in their last bits alone, negative ones and NaN"""
    p = K.Problem(2, [20000, 9000, 12000, 17001, 30, 16385], heads=1, kv=1, d=64, group=64, page=64, spare=6 * 220)
    w = torch.exp(3 * torch.randn(6, 1, p.columns * 64, generator=p.g))
    w[1] = 0.25
    w[2] = torch.where(torch.rand(w[2].shape, generator=p.g) < 0.9, 0.0, w[2])
    w[3] = 1 + torch.randint(0, 5000, w[3].shape, generator=p.g) * 2.0 ** -23
    w[5] = torch.where(torch.rand(w[5].shape, generator=p.g) < 0.2, math.nan, w[5] - 1)
    into = p.spare[:6 * 220].view(6, 220) if away else None
    more = dict(workspace=torch.zeros(0, dtype=torch.uint8, device="cuda")) if alone else {}
    assert ascq_gpu.kv_evict_workspace_size(p.gpu(ascq_gpu), p.table.cuda()) > 0
    _check_evict(ascq_gpu, p, w, keep, recent, into, **more)


@pytest.mark.parametrize("equal", [False, True])
def test_evict_many_parts(ascq_gpu, equal):
    """more parts of a selection than a wave has lanes, with ties all over them"""
    p = K.Problem(2, [600001, 540000], heads=1, kv=1, d=64, group=64, page=1024, spare=0)
    w = torch.rand(2, 1, p.columns * 1024, generator=p.g)
    if equal:
        w = (4 * w).round()
    _check_evict(ascq_gpu, p, w, 3001, 17, None)


def test_evict_bad_pages(ascq_gpu):
    """tokens on no page move as zeros, and nothing is written to a page that does not exist"""
    p = K.Problem(4, [60, 60], heads=1, kv=1, d=64, group=32, page=16, spare=8)
    cache = p.gpu(ascq_gpu)
    before = [x.clone() for x in cache]
    p.table[0, 1] = -1
    into = torch.tensor([[int(p.spare[0]), 1 << 29], [-1, int(p.spare[1])]]).int()
    w = torch.rand(2, 1, 64, generator=p.g)
    kept, n, _ = ascq_gpu.kv_evict(cache, p.table.cuda(), torch.tensor([60, 60]).int().cuda(), w.cuda(), 32, 4, into=into.cuda())
    assert n.tolist() == [32, 32]
    for which in range(4):
        want = before[which].cpu().clone()
        for b in range(2):
            for i, t in enumerate(kept[b, 0].tolist()):
                src, dst = int(p.table[b, t // 16]), int(into[b, i // 16])
                if 0 <= dst < want.shape[0]:
                    want[dst, 0, i % 16] = before[which][src, 0, t % 16].cpu() if src >= 0 else 0
        assert torch.equal(list(cache)[which].cpu().view(torch.uint8), want.view(torch.uint8))
