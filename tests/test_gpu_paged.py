"""The paged key / value cache (ops.PagedCache, kv_append, paged_attention, paged_decode) against its definition in 64
bits: element types, head layouts, lengths from one position, pages that end inside a tile, windows with visible first
tokens, idle slots, what must not be read (NaN in unused slots, infinities in hidden positions, page numbers outside
the pool), streams, graphs and pools past 4 GiB. Needs a gfx950 GPU."""
from __future__ import annotations

import pytest
import torch

from opentars_amd import _lib, ops
from opentars_amd.contract import OUT_BF16, OUT_FP32
from paged_data import E4M3, QT, Layer, bits, compare, empty_pool, put

pytestmark = pytest.mark.gpu

SENTINEL = 77.0


def prompt(layer, y_dtype=None, **kw):
    cache, q, table, lens, starts = layer.dev(ops)
    y = torch.full(layer.q.shape, SENTINEL, dtype=y_dtype or layer.qt, device="cuda")
    want, tol = layer.want(y.cpu(), **{k: v for k, v in kw.items() if k in ("scale", "window", "sinks")})
    got = ops.paged_attention(cache, q, table, lens, starts, y=y, **kw)
    assert got is y
    compare(got, want, tol)


def decode(layer, y_dtype=None, **kw):
    cache, q, table, lens, _ = layer.dev(ops)
    y = torch.full(layer.q.shape, SENTINEL, dtype=y_dtype or layer.qt, device="cuda")
    want, tol = layer.want(y.cpu(), **kw)
    compare(ops.paged_decode(cache, q, table, lens, y=y, **kw), want, tol)


# ------------------------------------------------------------------------------------------------ kv_append
@pytest.mark.parametrize("layout", ["hnd", "nhd", "mixed"])
@pytest.mark.parametrize("qt,cache", [("bf16", "same"), ("fp16", "same"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("hd,kv,page", [(128, 8, 16), (64, 1, 32), (256, 3, 64)])
def test_append_stores_the_rows_and_nothing_else(layout, qt, cache, hd, kv, page):
    lens, rows = [1, 40, 0, 17, 70, 5], [1, 33, 0, 1, 70, 9]        # the last has more new rows than positions
    layer = Layer(hd + page, lens, rows, kv, kv, hd, page=page, qt=qt, cache=cache, layout=layout, spare=2)
    g = torch.Generator().manual_seed(1)
    total = sum(rows) + 2
    wide = torch.randn(total, 2 * kv * hd + 32, generator=g).to(layer.qt)
    wide[3, 5], wide[4, 6], wide[5, 7], wide[6, 8] = float("nan"), float("inf"), 60000.0, -3e-6
    k, v = wide[:, :kv * hd], wide[:, kv * hd + 16:2 * kv * hd + 16]
    dev = layer.dev(ops)
    pools = []
    for pool, x, scale in ((layer.kpool, k, layer.kscale), (layer.vpool, v, layer.vscale)):
        want = pool.clone(memory_format=torch.preserve_format)
        first = 0
        for b, (n, r) in enumerate(zip(lens, rows)):
            for i in range(r):
                p = n - r + i
                if p < 0:
                    continue
                row = x[first + i].view(kv, hd)
                if scale is not None:
                    row = (row.float() / scale[:, None]).clamp(-448, 448)
                put(want, [layer.where[b][p]], [row.to(layer.ct)])
            first += r
        pools.append(want)
    w = wide.cuda()
    ops.kv_append(dev[0], w[:, :kv * hd], w[:, kv * hd + 16:2 * kv * hd + 16], dev[2], dev[3], dev[4])
    for got, want in zip((dev[0].k, dev[0].v), pools):
        a, b = bits(got.cpu()), bits(want)
        if layer.ct == E4M3:                                          # either NaN
            a, b = (torch.where((t & 0x7F) == 0x7F, 0x7F, t) for t in (a, b))
        assert torch.equal(a, b)


def test_append_one_row_per_sequence_with_idle_slots():
    lens = [1, 0, 33, 16, 0, 100]
    layer = Layer(3, lens, [1] * 6, 2, 2, 64)
    x = torch.randn(6, 256).to(torch.bfloat16).cuda()
    cache, _, table, n, _ = layer.dev(ops)
    before = cache.k.clone(), cache.v.clone()
    ops.kv_append(cache, x[:, :128], x[:, 128:], table, n)
    for b, length in enumerate(lens):
        if length:
            page, slot = layer.where[b][length - 1]
            before[0][page, :, slot] = x[b, :128].view(2, 64)
            before[1][page, :, slot] = x[b, 128:].view(2, 64)
    assert torch.equal(bits(cache.k), bits(before[0])) and torch.equal(bits(cache.v), bits(before[1]))


def test_append_takes_binary16_bits_and_every_e4m3_value():
    """int16 rows are binary16 bits; every finite e4m3 value times its scale comes back as itself."""
    kv, hd = 2, 128
    k, v = (t.cuda() for t in empty_pool(4, kv, 16, hd, E4M3))
    codes = torch.arange(256, dtype=torch.uint8)
    vals = codes.view(E4M3).float()
    scale = torch.tensor([0.5, 2.0])
    x = torch.stack([vals[:128], vals[128:]]).mul(scale[:, None]).reshape(1, 256).half()
    cache = ops.PagedCache(k, v, scale.cuda(), scale.cuda())
    ops.kv_append(cache, x.view(torch.int16).cuda(), x.view(torch.int16).cuda(),
                  torch.tensor([[2]], dtype=torch.int32).cuda(), torch.tensor([4], dtype=torch.int32).cuda())
    for pool in (k, v):
        got = pool.cpu().view(torch.uint8)[2, :, 3].reshape(-1)
        keep = (codes & 0x7F) != 0x7F
        assert torch.equal(got[keep], codes[keep]) and bool(((got & 0x7F) == 0x7F)[~keep].all())


# ------------------------------------------------------------------------------------------------ paged_attention
@pytest.mark.parametrize("qt,cache", [("bf16", "same"), ("fp16", "same"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("heads,kv,hd,page", [(4, 4, 64, 16), (16, 8, 128, 16), (6, 2, 128, 64), (4, 1, 256, 32),
                                              (7, 1, 64, 128)])
def test_prompt_rows_of_ragged_sequences(qt, cache, heads, kv, hd, page):
    lens, rows = [1, 16, 17, 0, 65, 130, 5, 200], [1, 16, 3, 0, 65, 40, 9, 1]
    prompt(Layer(hd + heads, lens, rows, heads, kv, hd, page=page, qt=qt, cache=cache, spare=3))


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (16, 4), (64, 1), (33, 70), (100, 16), (300, 5)])
@pytest.mark.parametrize("hd,qt,cache", [(128, "bf16", "same"), (64, "fp16", "e4m3"), (256, "fp16", "same")])
def test_prompt_rows_with_a_window_and_visible_first_tokens(window, sinks, hd, qt, cache):
    lens, rows = [260, 3, 129, 190], [150, 3, 1, 64]
    prompt(Layer(window + sinks, lens, rows, 4, 2, hd, qt=qt, cache=cache), window=window, sinks=sinks)


@pytest.mark.parametrize("layout", ["nhd", "mixed"])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_prompt_rows_over_other_strides(layout, cache):
    layer = Layer(9, [70, 33], [50, 2], 6, 3, 128, cache=cache, layout=layout, spare=1)
    cache_, q, table, lens, starts = layer.dev(ops)
    wide = torch.zeros(q.shape[0], q.shape[1] + 64, dtype=q.dtype, device="cuda")
    wide[:, 32:-32] = q
    y = torch.full((q.shape[0], q.shape[1] + 8), SENTINEL, device="cuda")
    want, tol = layer.want(y.cpu()[:, :q.shape[1]])
    tables = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    tables[:, :table.shape[1]] = table
    got = ops.paged_attention(cache_, wide[:, 32:-32], tables[:, :table.shape[1]], lens, starts, out=OUT_FP32,
                              y=y[:, :q.shape[1]])
    compare(got, want, tol)
    assert bool((y[:, q.shape[1]:] == SENTINEL).all())


@pytest.mark.parametrize("rows,past,heads,kv", [(1, 3000, 8, 2), (5, 2500, 16, 8), (33, 4100, 4, 1), (300, 700, 8, 8)])
def test_prompt_rows_over_longer_caches(rows, past, heads, kv):
    prompt(Layer(rows, [past + rows, past // 2 + rows], [rows, rows], heads, kv, 128, page=32), window=0)


@pytest.mark.parametrize("qt,cache", [("bf16", "same"), ("fp16", "same"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("heads,kv,hd,page", [(4, 4, 64, 16), (16, 4, 128, 16), (12, 2, 128, 64), (4, 1, 256, 32), (7, 1, 64, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 6)])
def test_few_rows_of_each_sequence(qt, cache, heads, kv, hd, page, window, sinks):
    """32 columns (rows times query heads of a K / V head) a sequence or fewer on average, some sequences with none, some
    with more."""
    rows = [1, 5, 0, 3, 40, 2, 1, 4, 0, 0, 1, 1, 0, 0, 2, 1, 1, 1, 1, 0]
    lens = [1, 70, 9, 500, 48, 1, 300, 4, 0, 55, 16, 17, 3, 0, 1000, 129, 128, 127, 33, 31]
    prompt(Layer(hd + heads, lens, rows, heads, kv, hd, page=page, qt=qt, cache=cache, spare=3), window=window, sinks=sinks)


@pytest.mark.parametrize("hd,kv", [(64, 2), (128, 8), (256, 1)])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_few_rows_over_split_lengths(hd, kv, cache):
    prompt(Layer(hd, [6000, 700, 3, 2500], [5, 6, 4, 7], 4 * kv, kv, hd, page=32, cache=cache))


def test_prompt_output_types_and_scale():
    layer = Layer(5, [50, 20], [31, 20], 4, 2, 64, spare=1)
    prompt(layer, torch.float32, scale=0.3)
    cache, q, table, lens, starts = layer.dev(ops)
    y = ops.paged_attention(cache, q, table, lens, starts, scale=0.3, out=OUT_FP32)
    assert y.dtype == torch.float32 and bool((y[51:] == 0).all())
    want, tol = layer.want(torch.zeros(y.shape), scale=0.3)
    compare(y, want, tol)
    assert ops.paged_attention(cache, q, table, lens, starts, out=OUT_BF16).dtype == torch.bfloat16
    half = Layer(5, [50, 20], [31, 20], 4, 2, 64, qt="fp16")
    cache, q, table, lens, starts = half.dev(ops)
    a = ops.paged_attention(cache, q, table, lens, starts)
    b = ops.paged_attention(cache, q.view(torch.int16), table, lens, starts)
    assert b.dtype == torch.int16 and torch.equal(a.view(torch.int16), b)


# ------------------------------------------------------------------------------------------------ paged_decode
@pytest.mark.parametrize("qt,cache", [("bf16", "same"), ("fp16", "same"), ("bf16", "e4m3"), ("fp16", "e4m3")])
@pytest.mark.parametrize("heads,kv,hd,page", [(8, 8, 64, 16), (16, 8, 128, 16), (3, 1, 128, 64), (4, 1, 256, 32),
                                              (20, 1, 128, 16), (64, 2, 64, 128), (40, 1, 256, 16)])
def test_decode_rows(qt, cache, heads, kv, hd, page):
    lens = [1, 0, 15, 16, 17, 33, 64, 65, 129, 300]
    decode(Layer(hd + heads, lens, [1] * len(lens), heads, kv, hd, page=page, qt=qt, cache=cache))


@pytest.mark.parametrize("lens,heads,kv,hd", [([5000], 8, 2, 128), ([9000, 3, 0, 2000], 4, 1, 64),
                                              ([1500] * 40, 4, 4, 128), ([4097, 4096, 4095], 16, 2, 256)])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_decode_rows_over_split_lengths(lens, heads, kv, hd, cache):
    decode(Layer(len(lens), lens, [1] * len(lens), heads, kv, hd, cache=cache))


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 70), (512, 4), (33, 1), (2000, 3)])
@pytest.mark.parametrize("hd,qt", [(128, "bf16"), (256, "fp16")])
def test_decode_with_a_window_and_visible_first_tokens(window, sinks, hd, qt):
    lens = [1300, 1, 0, 99, 100, 101, 533]
    decode(Layer(window, lens, [1] * len(lens), 4, 1, hd, qt=qt), window=window, sinks=sinks)


def test_decode_output_types():
    layer = Layer(2, [30, 500], [1, 1], 4, 2, 128)
    decode(layer, torch.float32)
    cache, q, table, lens, _ = layer.dev(ops)
    y = ops.paged_decode(cache, q, table, lens)
    assert y.dtype == torch.bfloat16
    compare(y, *layer.want(torch.zeros(y.shape, dtype=torch.bfloat16)))


def test_many_sequences():
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (1500,), generator=g).tolist()
    layer = Layer(1, lens, [1] * 1500, 2, 1, 64)
    decode(layer)
    rows = [min(n, 1 + i % 3) for i, n in enumerate(lens)]
    prompt(Layer(1, lens, rows, 2, 1, 64))


def test_prompts_of_many_sequences():
    """More sequences than a wave has lanes, some without rows."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 70, (150,), generator=g).tolist()
    rows = [0 if i % 7 == 3 else min(n, 20 + i % 30) for i, n in enumerate(lens)]
    prompt(Layer(2, lens, rows, 4, 1, 64, spare=3))


@pytest.mark.parametrize("heads,kv,hd,qt,cache", [(16, 4, 64, "fp16", "same"), (16, 2, 128, "bf16", "same"),
                                                  (6, 2, 128, "bf16", "e4m3"), (8, 2, 256, "bf16", "same"), (2, 2, 256, "fp16", "e4m3")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 3)])
def test_some_rows_behind_short_caches(heads, kv, hd, qt, cache, window, sinks):
    layer = Layer(21, [301, 77, 0, 290, 310, 5], [61, 77, 0, 1, 40, 9], heads, kv, hd, qt=qt, cache=cache, spare=2)
    prompt(layer, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
def test_more_tiles_than_run_at_once(window, sinks):
    """Prompts of several sequences that come to more workgroups than the GPU holds: they start in the order of their
    length."""
    rows = [3, 330, 0, 130, 64, 1, 210, 20, 0, 190, 65, 63]
    lens = [r + (37 * i) % 90 for i, r in enumerate(rows)]
    lens[4] = 40                                                        # more new rows than positions
    prompt(Layer(7, lens, rows, 64, 32, 64, spare=2), window=window, sinks=sinks)


def test_the_slices_of_a_long_batch_give_the_same_rows():
    """9000 sequences of up to 60 positions, five new rows each (none for some), stored and attended at once, and 30 at a
    time: no sequence is split here, so every row has the same bits."""
    seqs, kv, hd, group, page = 9000, 1, 64, 8, 16
    g = torch.Generator().manual_seed(6)
    lens = torch.randint(5, 61, (seqs,), generator=g, dtype=torch.int32)
    rows = torch.where(torch.arange(seqs) % 11 == 5, 0, 5)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), rows.cumsum(0)]).to(torch.int32)
    total = int(starts[-1])
    table = torch.randperm(4 * seqs, generator=g).to(torch.int32).view(seqs, 4).cuda()
    k, v = (torch.randn(4 * seqs, kv, page, hd, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    new, q = (torch.randn(total + 9, n, generator=g).to(torch.bfloat16).cuda() for n in (2 * kv * hd, group * hd))
    whole, parts = (ops.PagedCache(k.clone(), v.clone()) for _ in range(2))
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    z = y.clone()
    ld, sd = lens.cuda(), starts.cuda()
    ops.kv_append(whole, new[:, :hd], new[:, hd:], table, ld, sd)
    ops.paged_attention(whole, q, table, ld, sd, y=y)
    for b in list(range(0, 300, 30)) + list(range(4000, 4300, 30)) + list(range(seqs - 300, seqs, 30)):
        r0, r1 = int(starts[b]), int(starts[b + 30])
        ops.kv_append(parts, new[r0:r1, :hd], new[r0:r1, hd:], table[b:b + 30], ld[b:b + 30], sd[b:b + 31] - r0)
        ops.paged_attention(parts, q[r0:r1], table[b:b + 30], ld[b:b + 30], sd[b:b + 31] - r0, y=z[r0:r1])
        t = table[b:b + 30].flatten().long()
        assert torch.equal(bits(whole.k[t]), bits(parts.k[t])) and torch.equal(bits(whole.v[t]), bits(parts.v[t]))
        assert torch.equal(bits(y[r0:r1]), bits(z[r0:r1]))
    assert bool((y[total:] == SENTINEL).all())
    assert bool(torch.isfinite(y.float()).all()) and not bool((y[:total] == SENTINEL).all(1).any())


# ------------------------------------------------------------------------------------------------ what must not be read
@pytest.mark.parametrize("hd,cache", [(128, "same"), (64, "e4m3"), (256, "same")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 4)])
def test_hidden_positions_never_change_a_row(hd, cache, window, sinks):
    """Infinities and NaN in positions that a row does not see: ahead of it, or behind its window. Rows that see one are
    not finite in its columns; every other row is what it was."""
    lens, rows = [150], [150]
    layer = Layer(6, lens, rows, 4, 2, hd, qt="fp16", cache=cache)
    bad = {60: float("inf"), 61: float("nan"), 119: float("-inf")}
    for p, value in bad.items():
        page, slot = layer.where[0][p]
        for pool, col in ((layer.kpool, 3), (layer.vpool, 9)):
            if pool.dtype == E4M3:
                pool.view(torch.uint8)[page, 0, slot, col] = 0x7F
            else:
                pool[page, 0, slot, col] = value
    cache_, q, table, n, starts = layer.dev(ops)
    got = ops.paged_attention(cache_, q, table, n, starts, window=window, sinks=sinks, out=OUT_FP32).cpu()
    want, tol = layer.want(torch.zeros(got.shape), window=window, sinks=sinks)
    p = torch.arange(150)
    clean = torch.ones(150, dtype=torch.bool)
    for j in bad:
        clean &= ~((j <= p) & ((j > p - window) if window else True))
    assert int(clean.sum()) > 20
    compare(got[clean], want[clean], tol[clean])
    dirty = got[~clean][:, :2 * hd]                                    # the K / V head that holds them: 2 query heads
    assert not bool(torch.isfinite(dirty).all(1).any())
    compare(got[:, 2 * hd:], want[:, 2 * hd:], tol[:, 2 * hd:])        # the other K / V head's


@pytest.mark.parametrize("hd,cache", [(128, "same"), (64, "e4m3"), (256, "same"), (128, "e4m3")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
@pytest.mark.parametrize("n", [70, 1300])
def test_hidden_positions_never_change_one_of_few_rows(hd, cache, window, sinks, n):
    """The same for eight rows of a sequence, the hidden positions among their own, in one part and in several."""
    layer = Layer(7, [n, n], [8, 8], 4, 2, hd, qt="fp16", cache=cache)
    bad = {n - 3: float("inf"), n - 5: float("nan")}
    if window:
        bad[n - 27] = float("-inf")                                    # the first row's window alone holds it
    for p, value in bad.items():
        page, slot = layer.where[0][p]
        for pool, col in ((layer.kpool, 3), (layer.vpool, 9)):
            if pool.dtype == E4M3:
                pool.view(torch.uint8)[page, 0, slot, col] = 0x7F
            else:
                pool[page, 0, slot, col] = value
    cache_, q, table, lens, starts = layer.dev(ops)
    got = ops.paged_attention(cache_, q, table, lens, starts, window=window, sinks=sinks, out=OUT_FP32).cpu()
    want, tol = layer.want(torch.zeros(got.shape), window=window, sinks=sinks)
    p = torch.arange(n - 8, n)
    clean = torch.ones(8, dtype=torch.bool)
    for j in bad:
        clean &= ~((j <= p) & ((j > p - window) if window else True))
    assert int(clean.sum()) == (2 if window else 3)
    compare(got[:8][clean], want[:8][clean], tol[:8][clean])
    assert not bool(torch.isfinite(got[:8][~clean][:, :2 * hd]).all(1).any())
    compare(got[:, 2 * hd:], want[:, 2 * hd:], tol[:, 2 * hd:])
    compare(got[8:], want[8:], tol[8:])


def test_an_infinity_in_v_reaches_its_own_column_of_the_rows_that_see_it():
    """V alone holds an infinity, ahead of some rows: the rows that see it are infinite in its column and nowhere else."""
    for rows in (8, 100):
        layer = Layer(rows, [200], [rows], 4, 2, 64, qt="bf16")
        page, slot = layer.where[0][196]
        layer.vpool[page, 1, slot, 20] = float("inf")
        cache, q, table, lens, starts = layer.dev(ops)
        got = ops.paged_attention(cache, q, table, lens, starts, out=OUT_FP32).cpu()
        want, tol = layer.want(torch.zeros(got.shape))
        see = torch.arange(200 - rows, 200) >= 196
        cols = [2 * 64 + 20, 3 * 64 + 20]
        assert bool(torch.isposinf(got[see][:, cols]).all())
        rest = torch.ones(256, dtype=torch.bool)
        rest[cols] = False
        compare(got[:, rest], want[:, rest], tol[:, rest])
        compare(got[~see], want[~see], tol[~see])


@pytest.mark.parametrize("hd,cache", [(128, "same"), (64, "e4m3")])
def test_page_numbers_outside_the_pool_hold_nothing(hd, cache):
    lens, rows = [100, 50, 20], [40, 1, 20]
    layer = Layer(8, lens, rows, 4, 2, hd, cache=cache)
    layer.table[0, 1], layer.table[0, 4], layer.table[1, 0] = -5, 2 ** 31 - 1, layer.kpool.shape[0]
    layer.table[2, 0], layer.table[2, 1] = -1, -2 ** 31                # the third sequence has no page at all
    hidden = [(0, p) for p in range(100) if p // 16 in (1, 4)] + [(1, p) for p in range(16)] + [(2, p) for p in range(20)]
    cache_, q, table, n, starts = layer.dev(ops)
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    want, tol = layer.want(y.cpu(), hidden=hidden)
    compare(ops.paged_attention(cache_, q, table, n, starts, y=y), want, tol)
    layer.rows = [1, 1, 1]
    layer.q = layer.q[:3]
    y = torch.full((3, q.shape[1]), SENTINEL, dtype=q.dtype, device="cuda")
    want, tol = layer.want(y.cpu(), hidden=hidden)
    compare(ops.paged_decode(cache_, q[:3].contiguous(), table, n, y=y), want, tol)
    before = cache_.k.clone(), cache_.v.clone()
    x = torch.ones(3, 2 * hd, dtype=q.dtype, device="cuda")
    ops.kv_append(cache_, x, x, table, torch.tensor([80, 3, 20], dtype=torch.int32).cuda())   # every one on such a page
    assert torch.equal(bits(cache_.k), bits(before[0])) and torch.equal(bits(cache_.v), bits(before[1]))


def test_lengths_and_starts_out_of_range_are_clamped():
    """Lengths past the table, negative ones, starts that descend or pass the rows: the values stay inside the call's
    buffers. What the rows in range get is their definition with the clamped values."""
    layer = Layer(12, [64, 64], [4, 4], 2, 1, 64, width=4)
    cache, q, table, _, _ = layer.dev(ops)
    t = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    want, tol = layer.want(y.cpu())
    compare(ops.paged_attention(cache, q, table, t(1000, 2 ** 31 - 1), t(0, 4, 8), y=y), want, tol)
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    ops.paged_attention(cache, q, table, t(64, -3), t(-2, 4, 99), y=y)
    compare(y[:4], want[:4], tol[:4])
    assert bool((y[4:] == 0).all())
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    ops.paged_attention(cache, q, table, t(64, 64), t(6, 2, 2 ** 31 - 1), y=y)   # descends: the first has no rows
    torch.cuda.synchronize()
    assert bool((y[:2] == SENTINEL).all()) and bool(torch.isfinite(y.float()).all())
    before = cache.k.clone()
    ops.kv_append(cache, q[:2, :64], q[:2, :64], table, t(-5, 0))
    assert torch.equal(bits(cache.k), bits(before))


@pytest.mark.parametrize("seqs", [40, 200])
@pytest.mark.parametrize("rows", [1, 12, 40])
def test_starts_that_do_not_ascend_stay_inside_the_calls_buffers(seqs, rows):
    """Row spans that overlap come to more parts than the sizes allow for; what surrounds the buffers keeps its bits, and a
    right call after it its results."""
    layer = Layer(13, [1200] * 3, [rows] * 3, 4, 2, 64)
    cache, q, table, lens, _ = layer.dev(ops)
    table, lens = (t.repeat(seqs // 3 + 1, *[1] * (t.dim() - 1))[:seqs].contiguous() for t in (table, lens))
    q = q.repeat(seqs // 3 + 1, 1)[:rows * seqs].contiguous()
    good = torch.arange(seqs + 1, dtype=torch.int32).cuda() * rows
    want = ops.paged_attention(cache, q, table, lens, good).clone()
    around = torch.full((rows * seqs + 64, q.shape[1]), SENTINEL, dtype=q.dtype, device="cuda")
    y = around[32:32 + rows * seqs]
    before = cache.k.clone(), cache.v.clone()
    ends = torch.tensor([0, rows * seqs], dtype=torch.int32).repeat(seqs // 2 + 1)[:seqs + 1].cuda()
    for starts in (ends, good.flip(0), ends.flip(0), good * -3, good * 5 - 7):
        ops.paged_attention(cache, q, table, lens, starts.contiguous(), y=y)
        torch.cuda.synchronize()
        assert bool((around[:32] == SENTINEL).all()) and bool((around[32 + rows * seqs:] == SENTINEL).all())
    assert torch.equal(bits(cache.k), bits(before[0])) and torch.equal(bits(cache.v), bits(before[1]))
    assert torch.equal(bits(ops.paged_attention(cache, q, table, lens, good)), bits(want))


# ------------------------------------------------------------------------------------------------ how calls are made
def test_empty_calls_do_nothing():
    layer = Layer(1, [5], [5], 2, 1, 64)
    cache, q, table, lens, starts = layer.dev(ops)
    assert ops.paged_attention(cache, q[:0], table, lens, starts).shape == (0, 128)
    assert ops.paged_decode(cache, q[:0], table[:0], lens[:0]).shape == (0, 128)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    assert bool((ops.paged_attention(cache, q, table[:0], lens[:0], none, y=y) == SENTINEL).all())
    ops.kv_append(cache, q[:0, :64], q[:0, :64], table, lens, starts)
    ops.kv_append(cache, q[:, :64], q[:, :64], table[:0], lens[:0], none)


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("rows,heads,kv,hd", [
    ([1, 1, 1, 1], 8, 2, 128), ([4, 0, 0, 0], 24, 2, 64), ([0, 3, 0, 1], 12, 1, 128), ([9, 1, 17, 0], 8, 8, 64),
    ([6, 2, 5, 8], 16, 4, 256), ([40, 0, 90, 3], 8, 2, 64), ([200, 130, 1, 0], 4, 2, 128), ([70, 0, 0, 66], 6, 3, 256)])
def test_the_workspace_is_as_large_as_the_calls_use(rows, heads, kv, hd, window):
    """What lies behind it keeps its bits, however the rows are spread over the sequences."""
    layer = Layer(14, [2600, 700, 3300, 90], rows, heads, kv, hd)
    cache, q, table, lens, starts = layer.dev(ops)
    lib, n, stream = _lib.lib(), sum(rows), torch.cuda.current_stream().cuda_stream
    y = torch.full(q.shape, SENTINEL, dtype=q.dtype, device="cuda")
    for decode in [0, 1] if rows == [1, 1, 1, 1] else [0]:
        need = lib.tars_paged_workspace(heads, kv, hd, n, 4, table.shape[1], 16, decode)
        assert need % 16 == 0
        work = torch.full((need // 4 + 4096,), SENTINEL, device="cuda")
        args = (cache._ref, q.data_ptr(), 0, 0, heads, n, y.data_ptr(), 0, OUT_BF16, hd ** -0.5, window, 3, table.data_ptr(), 0,
                table.shape[1], lens.data_ptr())
        if decode:
            assert lib.tars_paged_decode(*args, work.data_ptr(), need, stream) == 0
        else:
            assert lib.tars_paged_attention(*args, starts.data_ptr(), 4, work.data_ptr(), need, stream) == 0
        assert bool((work[need // 4:] == SENTINEL).all())
        compare(y, *layer.want(torch.zeros(y.shape, dtype=y.dtype), window=window, sinks=3 if window else 0))


@pytest.mark.parametrize("decode", [0, 1])
def test_a_workspace_that_no_call_needs_is_left_alone(decode):
    layer = Layer(2, [40, 17], [1, 1], 2, 1, 64)
    cache, q, table, lens, starts = layer.dev(ops)
    assert _lib.lib().tars_paged_workspace(2, 1, 64, 2, 2, table.shape[1], 16, decode) == 0
    work = torch.full((64,), SENTINEL, device="cuda")
    y = torch.empty_like(q)
    args = (cache._ref, q.data_ptr(), 0, 0, 2, 2, y.data_ptr(), 0, OUT_BF16, 0.125, 0, 0, table.data_ptr(), 0, table.shape[1],
            lens.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    lib = _lib.lib()
    if decode:
        assert lib.tars_paged_decode(*args, work.data_ptr(), 0, stream) == 0
    else:
        assert lib.tars_paged_attention(*args, starts.data_ptr(), 2, work.data_ptr(), 0, stream) == 0
    compare(y, *layer.want(torch.zeros(y.shape, dtype=y.dtype), scale=0.125))
    assert bool((work == SENTINEL).all())


def test_rows_that_are_one_and_the_same_are_refused():
    """A broadcast row has no stride of its own, which a stride of 0 (dense) would read past; one row alone is fine."""
    layer = Layer(1, [5, 9, 7], [1, 1, 1], 2, 1, 64)
    cache, q, table, lens, starts = layer.dev(ops)
    same, pages = q[:1].expand(3, -1), table[:1].expand(3, -1)
    for call in (lambda: ops.paged_decode(cache, same, table, lens), lambda: ops.paged_decode(cache, q, pages, lens),
                 lambda: ops.paged_decode(cache, q, table, lens, y=same), lambda: ops.paged_decode(cache, q, table, lens[:1].expand(3)),
                 lambda: ops.paged_attention(cache, same, table, lens, starts),
                 lambda: ops.paged_attention(cache, q, table, lens, starts[:1].expand(4)),
                 lambda: ops.kv_append(cache, same[:, :64], q[:, :64], table, lens),
                 lambda: ops.kv_append(cache, q[:, :64], same[:, :64], table, lens),
                 lambda: ops.kv_append(cache, q[:, :64], q[:, :64], pages, lens)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        ops.paged_decode(cache, q[0], table, lens)
    want = ops.paged_decode(cache, q, table, lens)
    one = torch.as_strided(q, (1, q.shape[1]), (1, 1)), torch.as_strided(table, (1, table.shape[1]), (0, 1))   # any stride
    assert torch.equal(bits(ops.paged_decode(cache, *one, lens[:1])), bits(want[:1]))


def test_refusals_of_the_wrappers():
    layer = Layer(1, [5], [5], 4, 2, 64)
    cache, q, table, lens, starts = layer.dev(ops)
    k = cache.k
    with pytest.raises(ValueError):
        ops.PagedCache(k, k[:, :1])
    with pytest.raises(ValueError):
        ops.PagedCache(k, cache.v.half())
    with pytest.raises(ValueError):
        ops.PagedCache(k.cpu(), cache.v.cpu())
    with pytest.raises(ValueError):
        ops.PagedCache(k, cache.v, torch.ones(3, device="cuda"))
    with pytest.raises(ValueError):
        ops.PagedCache(k.float(), k.float())
    bad = [dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :64]), dict(table=table.long()), dict(lens=lens.long()),
           dict(lens=lens.cpu()), dict(starts=starts[:1]), dict(table=table.repeat(2, 1)), dict(y=q.float()[:2]),
           dict(out=OUT_FP32, y=torch.empty_like(q))]
    good = dict(q=q, table=table, lens=lens, starts=starts)
    for kw in bad:
        with pytest.raises(ValueError):
            ops.paged_attention(cache, **{**good, **kw})
    for kw, name in ((dict(scale=0.0), "E_FIELD"), (dict(scale=float("nan")), "E_FIELD"), (dict(window=-1), "E_FIELD"),
                     (dict(sinks=-1), "E_FIELD"), (dict(out=2), "E_FIELD"), (dict(q=q.half()), "E_FIELD")):
        with pytest.raises(ops.TarsError) as e:
            ops.paged_attention(cache, **{**good, **kw})
        assert e.value.name == name, kw
    with pytest.raises(ops.ContractError):
        ops.paged_attention(cache, **good, y=q)
    with pytest.raises(ops.TarsError):                                 # heads of 32
        ops.paged_decode(ops.PagedCache(k[..., :32], cache.v[..., :32]), q[:1, :128], table, lens)
    with pytest.raises(ops.ContractError):
        ops.kv_append(ops.PagedCache(k, k), q[:, :128], q[:, :128], table, lens, starts)
    with pytest.raises(ValueError):
        ops.kv_append(cache, q[:, :128], q[:, :64], table, lens, starts)
    with pytest.raises(ValueError):
        ops.paged_decode(cache, q, table, lens)


def test_another_stream():
    layer = Layer(21, [900, 40], [1, 1], 8, 2, 128)
    cache, q, table, lens, starts = layer.dev(ops)
    want, tol = layer.want(torch.zeros(q.shape, dtype=q.dtype))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = ops.paged_decode(cache, q, table, lens)
        b = ops.paged_attention(cache, q, table, lens, starts)
    c = ops.paged_decode(cache, q, table, lens)
    torch.cuda.synchronize()
    for y in (a, b, c):
        compare(y, want, tol)
    assert torch.equal(a, c)


def test_calls_on_two_streams_at_once():
    layers = [Layer(15 + i, [3000 + 500 * i, 40, 1500], [1, 1, 1], 8, 2, 128) for i in range(2)]
    prompts = [Layer(17 + i, [900, 2000], [5, 60 + i], 8, 2, 128) for i in range(2)]
    calls = [(*a.dev(ops), *b.dev(ops)) for a, b in zip(layers, prompts)]
    want = [(ops.paged_decode(*c[:4]), ops.paged_attention(*c[5:])) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append((ops.paged_decode(*c[:4]), ops.paged_attention(*c[5:])))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for pair in g:
            assert all(torch.equal(bits(x), bits(y)) for x, y in zip(w, pair))


def test_two_captured_graphs_replayed_between_eager_calls():
    """A decode step (store, attend) captured twice over two caches, replayed with lengths that grow on the device and
    eager calls between: each replay gives what the eager calls give at that length."""
    layers = [Layer(30 + i, [2000 + 300 * i, 10, 0, 77], [1] * 4, 8, 2, 128, cache=c, width=160, extra_pages=9)
              for i, c in enumerate(("same", "e4m3"))]
    calls = []
    for layer in layers:
        cache, q, table, lens, _ = layer.dev(ops)
        spare = [p for p in range(layer.kpool.shape[0]) if p not in set(table.flatten().tolist())]
        for b, n in enumerate(layer.lens):                             # a page for the positions to come
            table[b, -(-n // 16)] = spare[b]
        new = torch.randn(4, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
        calls.append((cache, q, table, lens, new, torch.zeros(q.shape, dtype=q.dtype, device="cuda")))

    def step(cache, q, table, lens, new, y):
        ops.kv_append(cache, new[:, :256], new[:, 256:], table, lens)
        ops.paged_decode(cache, q, table, lens, y=y)

    graphs = []
    for c in calls:
        step(*c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(*c)
        graphs.append(g)
    for t in range(4):
        got = []
        for g, c in zip(graphs, calls):
            c[3].add_(torch.tensor([1, 1, 0, 1], dtype=torch.int32).cuda())
            c[4].mul_(1.01)
            c[5].fill_(SENTINEL)
        for g in graphs:                                              # one behind the other, nothing waits between
            g.replay()
        for c in calls:
            got.append((c[5].clone(), bits(c[0].k).clone()))
        for (y, k), c in zip(got, calls):
            step(*c)
            torch.cuda.synchronize()
            assert torch.equal(y, c[5]) and torch.equal(k, bits(c[0].k)), t
            assert bool(torch.isfinite(y.float()).all()) and bool((y[2] == 0).all())


def test_pools_past_4_gib():
    kv, page, hd = 8, 64, 128
    pages = 34000                                                      # 131072 bytes each: 4.46 GB a pool
    k = torch.zeros(pages, kv, page, hd, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    cache = ops.PagedCache(k, v)
    layer = Layer(40, [200, 70], [200, 1], 8, 8, hd, page=page, extra_pages=0)
    far = torch.tensor([pages - 1, 5, 32768, pages - 7, 33333, 1], dtype=torch.int32)
    table = far.view(2, 3).repeat_interleave(1, 0)
    table = torch.stack([torch.cat([far[:4], far[:1]]), torch.cat([far[4:], far[:3]])]).contiguous().cuda()
    lens = torch.tensor([200, 70], dtype=torch.int32).cuda()
    starts = torch.tensor([0, 200, 270], dtype=torch.int32).cuda()
    rows = [torch.cat([x[0], x[1]]).reshape(270, kv * hd).to(torch.bfloat16).cuda() for x in (layer.K, layer.V)]
    ops.kv_append(cache, *rows, table, lens, starts)
    assert torch.equal(k[pages - 1, :, 0].reshape(-1), rows[0][0]) and torch.equal(v[1, :, 5].reshape(-1), rows[1][269])
    want, tol = layer.want(torch.zeros(201, 1024, dtype=torch.bfloat16))
    q = layer.q.cuda()
    compare(ops.paged_attention(cache, q, table, lens, torch.tensor([0, 200, 201], dtype=torch.int32).cuda()), want, tol)
    compare(ops.paged_decode(cache, q[[199, 200]].contiguous(), table, lens), want[[199, 200]], tol[[199, 200]])


def test_a_layer_from_quantized_linears_to_the_cache_and_back():
    """A decoder layer's attention as the framework's ops make it: W8A8 q / k / v, RoPE to bf16, the cache, attention in
    fp32, the per-token quantizer and the output projection: a prompt, then single tokens, against the dense
    definition over the very bf16 rows that were stored."""
    heads, kv, hd, H = 8, 2, 64, 512
    g = torch.Generator().manual_seed(11)
    W = {n: torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8).cuda()
         for n, rows, cols in (("q", heads * hd, H), ("k", kv * hd, H), ("v", kv * hd, H), ("o", H, heads * hd))}
    s = {n: (1e-4 + 2e-4 * torch.rand(w.shape[0], generator=g)).cuda() for n, w in W.items()}
    k, v = (t.cuda() for t in empty_pool(12, kv, 16, hd, torch.bfloat16))
    cache = ops.PagedCache(k, v)
    table = torch.tensor([[7, 2, 9, 0, 11, 4]], dtype=torch.int32).cuda()
    ang = torch.arange(96)[:, None] / 1e4 ** (torch.arange(0, hd, 2)[None] / hd)
    tab = torch.cat([ang.cos(), ang.sin()], 1).float().cuda()
    seen = {"k": [], "v": []}
    done = 0
    for rows in (37, 1, 1, 5):
        x = torch.randn(rows, H, generator=g).cuda()
        qf, kf, vb = ops.quant_gemm_rowcol(x, [(W["q"], s["q"]), (W["k"], s["k"]), (W["v"], s["v"], None, 0, OUT_BF16)])
        at = tab[done:done + rows].contiguous()
        qb = ops.rope_rows(qf.view(-1, hd), at, heads, hd, out=OUT_BF16).view(rows, -1)
        kb = ops.rope_rows(kf.view(-1, hd), at, kv, hd, out=OUT_BF16).view(rows, -1)
        done += rows
        lens = torch.tensor([done], dtype=torch.int32).cuda()
        starts = None if rows == 1 else torch.tensor([0, rows], dtype=torch.int32).cuda()
        ops.kv_append(cache, kb, vb, table, lens, starts)
        y = (ops.paged_decode(cache, qb, table, lens, out=OUT_FP32) if rows == 1 else
             ops.paged_attention(cache, qb, table, lens, starts, out=OUT_FP32))
        qq, sq = ops.quant_rows(y)
        z = ops.gemm_rowcol(qq, sq, W["o"], s["o"])
        assert z.shape == (rows, H) and bool(torch.isfinite(z).all())
        seen["k"].append(kb.cpu().double().view(rows, kv, hd))
        seen["v"].append(vb.cpu().double().view(rows, kv, hd))
        dense = Layer(0, [done], [rows], heads, kv, hd)
        dense.q, dense.K, dense.V = qb.cpu(), [torch.cat(seen["k"])], [torch.cat(seen["v"])]
        compare(y, *dense.want(torch.zeros(y.shape)))
