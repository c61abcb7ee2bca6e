"""The norm and rotation of queries and keys on the GPU (ops.qk_norm_rope, kv_append_rope) against their definition in 64 bits,
and kv_append_rope against the calls that it joins. Needs a gfx950 GPU."""
from __future__ import annotations

import math

import pytest
import torch

from opentars_amd import ops
from paged_data import E4M3, QT, Layer, bits
from step_data import HALF, TINY, rotated, table

pytestmark = pytest.mark.gpu


def positions(lens, rows):
    """(row, position) of the packed rows that have one."""
    out, first = [], 0
    for n, r in zip(lens, rows):
        out += [(first + i, n - r + i) for i in range(r) if n - r + i >= 0]
        first += r
    return out


def case(seed, lens, rows, heads, kv, hd, rot, qt, spare=2, norm=True):
    g = torch.Generator().manual_seed(seed)
    total = sum(rows) + spare
    fused = (2 * torch.randn(total, (heads + 2 * kv) * hd + 16, generator=g)).to(QT[qt])
    gam = 1 + 0.3 * torch.randn(2, hd, generator=g) if norm else (None, None)
    tab = table(max(lens) + 1, rot)
    starts = torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32)
    return fused, gam, tab, torch.tensor(lens, dtype=torch.int32), starts


def split(fused, heads, kv, hd):
    return fused[:, :heads * hd], fused[:, heads * hd:(heads + kv) * hd], fused[:, (heads + kv) * hd:(heads + 2 * kv) * hd]


def check(got, before, x, gamma, tab, at, hd, eps=1e-6):
    want, tol = before.double().clone(), torch.zeros(before.shape, dtype=torch.float64)
    if at:
        r, p = (torch.tensor(v) for v in zip(*at))
        y, t = rotated(x[r], gamma, tab, p, hd, eps)
        want[r] = y.flatten(1)
        tol[r] = (t + HALF[before.dtype] * (y.abs() + t) + TINY[before.dtype]).flatten(1)
    far = (got.cpu().double() - want).abs() - tol
    assert (far <= 0).all(), float(far.max())


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("qt", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv,hd,rot", [(16, 8, 128, 128), (1, 1, 64, 64), (3, 3, 64, 32), (8, 4, 256, 64), (5, 1, 256, 256),
                                             (40, 8, 128, 32), (7, 1, 64, 16), (2, 2, 128, 112)])
def test_packed_rows(qt, heads, kv, hd, rot):
    lens, rows = [1, 40, 0, 17, 300, 5], [1, 33, 0, 1, 20, 9]          # the last has more rows than positions
    fused, gam, tab, n, starts = case(heads + rot, lens, rows, heads, kv, hd, rot, qt)
    q, k, _ = split(fused, heads, kv, hd)
    yq, yk = torch.full(q.shape, 7.0, dtype=q.dtype), torch.full(k.shape, 7.0, dtype=q.dtype)
    qd, kd, _ = split(fused.cuda(), heads, kv, hd)
    gq, gk = ops.qk_norm_rope(qd, kd, hd, *cuda(tab, n, starts, *gam), yq=yq.cuda(), yk=yk.cuda())
    at = positions(lens, rows)
    check(gq, yq, q, gam[0], tab, at, hd)
    check(gk, yk, k, gam[1], tab, at, hd)


@pytest.mark.parametrize("norm", ["both", "none", "q", "k"])
def test_a_norm_of_one_or_none(norm):
    lens = [4, 9]
    fused, gam, tab, n, starts = case(1, lens, [4, 3], 4, 2, 64, 64, "bf16")
    qg, kg = gam[0] if norm in ("both", "q") else None, gam[1] if norm in ("both", "k") else None
    q, k, _ = split(fused, 4, 2, 64)
    qd, kd, _ = split(fused.cuda(), 4, 2, 64)
    gq, gk = ops.qk_norm_rope(qd, kd, 64, *cuda(tab, n, starts, qg, kg), eps=0.1)
    at = positions(lens, [4, 3])
    check(gq, torch.zeros(q.shape, dtype=q.dtype), q, qg, tab, at, 64, 0.1)
    check(gk, torch.zeros(k.shape, dtype=k.dtype), k, kg, tab, at, 64, 0.1)


def test_one_row_each_in_place_and_positions_behind_the_table():
    lens = [1, 0, 33, 16, 0, 100, 101]
    fused, gam, tab, n, _ = case(2, lens, [1] * 7, 4, 2, 128, 128, "fp16", spare=0)
    tab = tab[:100]                                                       # position 100 is not in it
    f = fused.cuda()
    q, k, v = split(f, 4, 2, 128)
    gq, gk = ops.qk_norm_rope(q, k, 128, *cuda(tab, n, None, *gam), yq=q, yk=k)
    assert gq is q and gk is k
    at = [(b, length - 1) for b, length in enumerate(lens) if 0 < length <= 100]
    q0, k0, v0 = split(fused, 4, 2, 128)
    check(gq, q0, q0, gam[0], tab, at, 128)
    check(gk, k0, k0, gam[1], tab, at, 128)
    assert torch.equal(v.cpu(), v0) and torch.equal(f[:, -16:].cpu(), fused[:, -16:])


def test_whatever_the_device_arrays_hold():
    """Starts that do not ascend, lengths below zero and past 2^30: nothing outside is written, and calls end."""
    fused, gam, tab, _, _ = case(3, [50], [40], 2, 1, 64, 64, "bf16")
    f = fused.cuda()
    q, k, _ = split(f, 2, 1, 64)
    for lens, starts in (([-5, 2 ** 31 - 1, 7], [0, 30, 10, 42]), ([9, 9, 9], [-3, 99, -7, 2 ** 31 - 1]), ([3, 3, 3], [5, 5, 5, 5])):
        room = torch.full((44, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        yq, _ = ops.qk_norm_rope(q, k, 64, *cuda(tab, torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32), *gam),
                                 yq=room[1:43])
        assert (room[0] == 7).all() and (room[43] == 7).all()


@pytest.mark.parametrize("qt,cache", [("bf16", "same"), ("fp16", "same"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("layout,heads,kv,hd,rot,page", [("hnd", 16, 8, 128, 128, 16), ("nhd", 3, 1, 64, 32, 32), ("mixed", 6, 3, 256, 64, 64)])
def test_into_the_cache(qt, cache, layout, heads, kv, hd, rot, page):
    lens, rows = [1, 40, 0, 17, 70, 5], [1, 33, 0, 1, 70, 9]
    layer = Layer(hd, lens, rows, heads, kv, hd, page=page, qt=qt, cache=cache, layout=layout, spare=2)
    fused, gam, tab, n, starts = case(4, lens, rows, heads, kv, hd, rot, qt)
    fused[3, (heads + kv) * hd + 5] = math.inf                            # a value
    fused[4, (heads + kv) * hd + 6] = math.nan
    handle, _, tb, ln, st = layer.dev(ops)
    before = [handle.k.cpu(), handle.v.cpu()]
    q, k, v = split(fused, heads, kv, hd)
    qd, kd, vd = split(fused.cuda(), heads, kv, hd)
    yq = torch.full(q.shape, 7.0, dtype=q.dtype)
    got = ops.kv_append_rope(handle, qd, kd, vd, tb, ln, tab.cuda(), st, *cuda(*gam), yq=yq.cuda())
    at = positions(lens, rows)
    check(got, yq, q, gam[0], tab, at, hd)
    # the values are kv_append's, to the bit
    other = layer.dev(ops)
    ops.kv_append(other[0], kd, vd, tb, ln, st)
    assert torch.equal(bits(handle.v.cpu()), bits(other[0].v.cpu()))
    # the keys: the definition's, rounded once; every other slot as it was
    place = {}
    first = 0
    for b, (length, r) in enumerate(zip(lens, rows)):
        for i in range(r):
            if length - r + i >= 0:
                place[first + i] = layer.where[b][length - r + i]
        first += r
    kk = handle.k.cpu()
    r, p = (torch.tensor(x) for x in zip(*at))
    want, tol = rotated(k[r], gam[1], tab, p, hd, 1e-6)
    for i, row in enumerate(r.tolist()):
        pg, slot = place[row]
        stored = kk[pg, :, slot]
        if cache == "e4m3":
            s = layer.kscale.double()[:, None]
            w = (want[i] / s).clamp(-448, 448)
            t = tol[i] / s + 2.0 ** -23 * w.abs()
            t = t + 2.0 ** -4 * (w.abs() + t) + 2.0 ** -10
        else:
            w, t = want[i], tol[i] + HALF[QT[qt]] * (want[i].abs() + tol[i]) + TINY[QT[qt]]
        assert ((stored.double() - w).abs() <= t).all()
        kk.view(torch.uint8 if kk.dtype == E4M3 else torch.int16)[pg, :, slot] = bits(before[0])[pg, :, slot]
    assert torch.equal(bits(kk), bits(before[0]))


@pytest.mark.parametrize("qt", ["bf16", "fp16"])
def test_into_the_cache_is_the_two_calls_joined(qt):
    """To the bit, for a pool of the rows' own type: the keys are rounded once either way."""
    lens, rows = [300, 7, 129], [130, 7, 1]
    layer = Layer(5, lens, rows, 8, 2, 128, qt=qt, spare=1)
    fused, gam, tab, n, starts = case(6, lens, rows, 8, 2, 128, 64, qt, spare=1)
    q, k, v = split(fused.cuda(), 8, 2, 128)
    one, two = layer.dev(ops), layer.dev(ops)
    t, gq, gk = cuda(tab, *gam)
    yq = ops.kv_append_rope(one[0], q, k, v, one[2], one[3], t, one[4], gq, gk)
    zq, zk = ops.qk_norm_rope(q, k, 128, t, two[3], two[4], gq, gk)
    ops.kv_append(two[0], zk, v, two[2], two[3], two[4])
    assert torch.equal(bits(yq), bits(zq)) and torch.equal(bits(one[0].k), bits(two[0].k)) and torch.equal(bits(one[0].v), bits(two[0].v))


def test_pages_and_positions_that_are_not_there():
    """A page number outside the pool, an idle slot, a position behind the table: neither key nor value is stored."""
    lens = [20, 0, 33, 50]
    layer = Layer(7, lens, [1] * 4, 2, 1, 64)
    fused, gam, tab, _, _ = case(8, lens, [1] * 4, 2, 1, 64, 64, "bf16", spare=0)
    cache, _, tb, ln, _ = layer.dev(ops)
    tb[2, 32 // 16] = 2 ** 30
    before = cache.k.clone(), cache.v.clone()
    q, k, v = split(fused.cuda(), 2, 1, 64)
    ops.kv_append_rope(cache, q, k, v, tb, ln, tab[:49].cuda(), None, *cuda(*gam))
    page, slot = layer.where[0][19]
    for pool, old in zip((cache.k, cache.v), before):
        changed = (bits(pool) != bits(old)).nonzero()
        assert len(changed) and set(map(tuple, changed[:, [0, 2]].tolist())) == {(page, slot)}


@pytest.mark.parametrize("decode", [True, False])
def test_streams_and_graphs(decode):
    lens, rows = ([30, 77], [1, 1]) if decode else ([40, 90], [40, 23])
    layer = Layer(9, lens, rows, 4, 2, 64)
    fused, gam, tab, _, _ = case(10, lens, rows, 4, 2, 64, 64, "bf16", spare=0)
    other = case(11, lens, rows, 4, 2, 64, 64, "bf16", spare=0)[0].cuda()
    t, gq, gk = cuda(tab, *gam)
    buf = fused.cuda()
    cache, _, tb, ln, st = layer.dev(ops)
    st = None if decode else st
    eager = []
    for x in (fused.cuda(), other):
        c = layer.dev(ops)[0]
        eager.append((ops.kv_append_rope(c, *split(x, 4, 2, 64), tb, ln, t, st, gq, gk), c.k, c.v))
    y = torch.zeros_like(eager[0][0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_append_rope(cache, *split(buf, 4, 2, 64), tb, ln, t, st, gq, gk, yq=y)
    for i in (1, 0, 1, 0):
        buf.copy_((fused.cuda(), other)[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(y), bits(eager[i][0])) and torch.equal(bits(cache.k), bits(eager[i][1])) and torch.equal(bits(cache.v), bits(eager[i][2]))


def test_refusals():
    fused, gam, tab, n, starts = cuda(*(lambda c: (c[0], None, c[2], c[3], c[4]))(case(1, [8, 8], [4, 4], 4, 2, 64, 64, "bf16")))
    q, k, v = split(fused, 4, 2, 64)
    for args, kw in (((q, k, 32, tab, n, starts), {}), ((q, k.half(), 64, tab, n, starts), {}), ((q.float(), k.float(), 64, tab, n, starts), {}),
                     ((q, k, 64, tab[:, :24].contiguous(), n, starts), {}), ((q, k, 64, tab.double(), n, starts), {}),
                     ((q, k, 64, tab, n.long(), starts), {}), ((q, k, 64, tab, n), {}), ((q, k, 64, tab, n, starts[:2]), {}),
                     ((q, k, 64, tab, n, starts), dict(qgamma=torch.zeros(63, device="cuda"))), ((q, k, 64, tab, n, starts), dict(eps=-1.0)),
                     ((q, k, 64, tab, n, starts), dict(eps=math.nan)), ((q, k, 64, tab, n, starts), dict(yq=q[:, 8:])),
                     ((q, k, 64, tab, n, starts), dict(yk=v[:, :64])), ((q, k, 64, tab, n, starts), dict(yk=q[:, :128])),
                     ((q, k, 64, torch.cat([tab, tab], 1), n, starts), {}), ((q, k[:-1], 64, tab, n, starts), {}), ((q, k, 64, tab.cpu(), n, starts), {})):
        with pytest.raises((ValueError, ops.TarsError)):
            ops.qk_norm_rope(*args, **kw)
