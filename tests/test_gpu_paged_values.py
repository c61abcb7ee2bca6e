"""Infinities and NaN in the paged cache that rows do see: they reach their own column of those rows, as the definition's
positive weights take them there, and change nothing else. Needs a gfx950 GPU."""
from __future__ import annotations

import pytest
import torch

from opentars_amd import ops
from opentars_amd.contract import OUT_FP32
from paged_data import E4M3, Layer, compare

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def plant(layer, b, p, head, col, value):
    """V of sequence b's position p, K / V head `head`: one value."""
    page, slot = layer.where[b][p]
    if layer.ct == E4M3:
        layer.vpool.view(torch.uint8)[page, head, slot, col] = 0x7F
    else:
        layer.vpool[page, head, slot, col] = value


def check(got, layer, planted, window=0, sinks=0, hidden=(), scale=None):
    """planted: (sequence, position, K / V head, column, value). The columns that hold one are the sum of those that the
    row sees; everything else is the definition's."""
    got = got.cpu()
    want, tol = layer.want(torch.zeros(got.shape, dtype=got.dtype), scale=scale, window=window, sinks=sinks, hidden=hidden)
    group, hd = layer.heads // layer.kv, layer.hd
    extra = torch.zeros(got.shape, dtype=got.dtype)
    first = 0
    for b, (n, r) in enumerate(zip(layer.lens, layer.rows)):
        for i in range(r):
            for s, p, head, col, value in planted:
                if s == b and p <= n - r + i and (not window or p > n - r + i - window or p < sinks):
                    extra[first + i, torch.arange(head * group, (head + 1) * group) * hd + col] += value
        first += r
    bad = extra != 0
    same = (got == extra) | (got.isnan() & extra.isnan())
    wrong = torch.nonzero(bad & ~same)
    assert not len(wrong), "%d of %d, the first at %s: %s, not %s" % (len(wrong), bad.sum(), wrong[0].tolist(), got[tuple(wrong[0])],
                                                                     extra[tuple(wrong[0])])
    compare(torch.where(bad, 0.0, got), torch.where(bad, 0.0, want), torch.where(bad, 1.0, tol))
    return int(bad.sum())


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("hd,qt,cache", [(64, "fp16", "same"), (128, "bf16", "same"), (128, "bf16", "e4m3"), (256, "bf16", "same")])
@pytest.mark.parametrize("rows", [8, 100])
@pytest.mark.parametrize("n", [300, 700])
def test_beside_a_page_outside_the_pool(n, rows, hd, qt, cache, value):
    """A value that every row sees, in a step whose other page is not in the pool: few rows and prompts, in one part and
    in several."""
    value = NAN if cache == "e4m3" or hd == 256 else value
    layer = Layer(n + rows, [n, 90], [rows, 3], 4, 2, hd, qt=qt, cache=cache)
    plant(layer, 0, 70, 1, 20, value)
    layer.table[0, 5] = -1                                             # positions 80 .. 95; 64 .. 95 are one step
    cache_, q, table, lens, starts = layer.dev(ops)
    got = ops.paged_attention(cache_, q, table, lens, starts, out=OUT_FP32)
    assert check(got, layer, [(0, 70, 1, 20, value)], hidden=[(0, p) for p in range(80, 96)]) == 2 * rows


SHAPES = [(64, "fp16", "same"), (128, "bf16", "same"), (128, "fp16", "e4m3"), (256, "bf16", "same"), (64, "bf16", "e4m3"),
          (256, "fp16", "same")]


def run(layer, decode, dtype, **kw):
    cache, q, table, lens, starts = layer.dev(ops)
    y = torch.empty(layer.q.shape, dtype=dtype, device="cuda")
    return ops.paged_decode(cache, q, table, lens, y=y, **kw) if decode else ops.paged_attention(cache, q, table, lens, starts, y=y, **kw)


@pytest.mark.parametrize("hd,qt,cache", SHAPES)
@pytest.mark.parametrize("n", [30, 300, 3000])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 5)])
def test_decode_gives_each_column_its_infinities(n, hd, qt, cache, window, sinks):
    """First, last and middle positions, in one part and in several; two of one sign in a column, and of both."""
    lens = [n, 1, n - 3]
    layer = Layer(n + hd, lens, [1, 1, 1], 6, 2, hd, qt=qt, cache=cache)
    planted = [(0, 0, 0, 3, INF), (0, n - 1, 1, 4, -INF), (0, n // 2, 0, 9, NAN), (0, n - 2, 0, 30, INF), (0, n - 9, 0, 30, INF),
               (0, n - 2, 0, 31, INF), (0, n - 9, 0, 31, -INF), (2, n - 4, 1, hd - 1, -INF), (2, 7, 1, 0, INF)]
    planted = [(*x, NAN if cache == "e4m3" else v) for *x, v in planted]
    for x in planted:
        plant(layer, *x)
    for dtype in (torch.float32, layer.qt):
        got = run(layer, True, dtype, window=window, sinks=sinks)
        assert check(got, layer, planted, window=window, sinks=sinks) >= 15   # five of the columns at least, three heads each


@pytest.mark.parametrize("hd,qt,cache", SHAPES)
@pytest.mark.parametrize("rows", [3, 8, 100])
@pytest.mark.parametrize("n", [300, 3000])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 5)])
def test_rows_give_each_column_its_infinities(n, rows, hd, qt, cache, window, sinks):
    """The same wherever the position stands: one that every row sees, one of the rows' own, one that leaves the window."""
    layer = Layer(n + rows + hd, [n, 40], [rows, 2], 4, 2, hd, qt=qt, cache=cache)
    planted = [(0, 2, 0, 3, INF), (0, n - rows - 20, 1, 4, -INF), (0, n - 2, 0, 9, INF), (0, n - 151, 1, 20, INF), (0, n - 170, 0, 21, NAN),
               (0, n - rows - 33, 0, 30, INF), (0, n - 1, 0, 30, -INF), (1, 38, 1, hd - 1, -INF)]
    planted = [(*x, NAN if cache == "e4m3" else v) for *x, v in planted]
    for x in planted:
        plant(layer, *x)
    for dtype in (torch.float32, layer.qt):
        got = run(layer, False, dtype, window=window, sinks=sinks)
        assert check(got, layer, planted, window=window, sinks=sinks) > 6 * rows


@pytest.mark.parametrize("hd,qt,cache", SHAPES)
@pytest.mark.parametrize("rows,n", [(1, 300), (1, 4000), (4, 300), (4, 4000), (100, 300), (100, 4000)])
def test_weights_too_small_for_fp32_are_positive(rows, n, hd, qt, cache):
    """One position outweighs all others by more than 2^150: the others' numerators, and the weights of the parts without
    it, round to 0, and an infinity beside them is one all the same."""
    layer = Layer(rows + n + hd, [n], [rows], 4, 2, hd, qt=qt, cache=cache)
    u = torch.randn(hd, generator=torch.Generator().manual_seed(3)).sign() * 1.5
    layer.q[:] = u.to(layer.qt).repeat(layer.heads)
    loud, k = n - rows - 100, 10.0 * u
    k = (k / layer.kscale[:, None]).clamp(-448, 448) if cache == "e4m3" else k.repeat(2, 1)
    k = k.to(layer.ct)
    page, slot = layer.where[0][loud]
    layer.kpool.view(torch.uint8 if cache == "e4m3" else layer.ct)[page, :, slot] = k.view(torch.uint8) if cache == "e4m3" else k
    layer.K[0][loud] = k.double() if cache != "e4m3" else k.double() * layer.kscale.double()[:, None]
    s = 0.4 * (layer.K[0].transpose(0, 1) @ layer.q[0, :hd].double())
    assert float(s[:, loud].min() - s[:, torch.arange(n) != loud].max()) > 105              # e^-105 < 2^-150
    planted = [(0, 5, 0, 3, INF), (0, 40, 1, 4, -INF), (0, loud - 3, 0, 9, NAN), (0, loud, 1, 30, INF)]
    planted = [(*x, NAN if cache == "e4m3" else v) for *x, v in planted]
    for x in planted:
        plant(layer, *x)
    got = run(layer, rows == 1, torch.float32, scale=0.4)
    assert check(got, layer, planted, scale=0.4) == 8 * rows


@pytest.mark.parametrize("rows,n", [(1, 300), (1, 4000), (4, 300), (4, 4000), (100, 300), (100, 4000)])
@pytest.mark.parametrize("hd,qt", [(64, "fp16"), (128, "bf16"), (256, "bf16")])
def test_a_nan_in_k_is_the_rows_result(rows, n, hd, qt):
    """A row that sees a NaN among its scores is NaN in every column, those with an infinity of V among them; the other K / V
    head is not touched."""
    layer = Layer(rows + n, [n], [rows], 4, 2, hd, qt=qt)
    page, slot = layer.where[0][33]
    layer.kpool[page, 0, slot, 7] = NAN
    plant(layer, 0, 50, 0, 3, INF)
    plant(layer, 0, 50, 1, 4, INF)
    for dtype in (torch.float32, layer.qt):
        got = run(layer, rows == 1, dtype).cpu()
        assert bool(got[:, :2 * hd].isnan().all())
        got[:, :2 * hd] = 0
        want, tol = layer.want(torch.zeros(got.shape, dtype=dtype))
        want[:, :2 * hd] = 0
        cols = torch.arange(2, 4) * hd + 4
        assert bool((got[:, cols] == INF).all())
        got[:, cols], want[:, cols] = 0, 0
        compare(got, want, tol)


# ------------------------------------------------------------------------------------------------ scales
@pytest.mark.parametrize("rows,n", [(1, 40), (1, 300), (1, 4000), (4, 300), (4, 4000), (100, 300), (100, 4000)])
@pytest.mark.parametrize("hd,qt", [(64, "fp16"), (128, "bf16"), (256, "bf16")])
def test_a_scale_that_fp32_rounds_to_nothing(rows, n, hd, qt):
    """scale times kscale is 1e-50: every visible position counts the same, hidden ones nothing."""
    layer = Layer(rows + n, [n], [rows], 4, 2, hd, qt=qt, cache="e4m3")
    layer.kscale[:] = 1e-20
    got = run(layer, rows == 1, torch.float32, scale=1e-30)
    compare(got, *layer.want(torch.zeros(got.shape), scale=1e-30))


@pytest.mark.parametrize("rows,n", [(1, 40), (1, 300), (1, 4000), (4, 300), (4, 4000), (100, 300), (100, 4000)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_a_scale_that_takes_scores_past_fp32(rows, n, hd, cache):
    """Scores of 1e40 and more: the largest has all the weight, so a row is V at that position."""
    layer = Layer(rows + n + hd, [n], [rows], 4, 2, hd, qt="bf16", cache=cache)
    u = torch.randn(hd, generator=torch.Generator().manual_seed(3)).sign() * 1e6
    layer.q[:] = u.to(layer.qt).repeat(layer.heads)
    loud = n - rows - 17
    page, slot = layer.where[0][loud]
    if cache == "e4m3":                                                # of 1e6 hd 448 and 3e38
        layer.kpool.view(torch.uint8)[page, :, slot] = (u.sign() * 448).to(E4M3).view(torch.uint8)
        layer.kscale[:] = 1e10
    else:
        layer.kpool[page, :, slot] = u.to(layer.qt)
    got = run(layer, rows == 1, torch.float32, scale=1e30).cpu().double()
    want = layer.V[0][loud].repeat_interleave(2, 0).reshape(1, -1).expand(rows, -1)
    assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs()).all())  # the scale's product, a reciprocal of 1


@pytest.mark.parametrize("rows,n", [(1, 300), (1, 4000), (4, 700), (100, 300), (100, 4000)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_mean_of_binary16_values_is_in_their_range(rows, n, hd):
    """Columns of V that hold binary16's largest value at every position: so does every row, however its numerators are
    rounded (a part in 2^12 more is an infinity)."""
    layer = Layer(rows + n + hd, [n], [rows], 4, 2, hd, qt="fp16")
    layer.q *= 8                                                       # one position or two have most of the weight
    for page, slot in layer.where[0]:
        layer.vpool[page, 0, slot, ::2], layer.vpool[page, 1, slot, 1::2] = 65504.0, -65504.0
    got = run(layer, rows == 1, torch.float16).cpu()
    got = got.view(rows, 2, 2, hd)
    assert bool(torch.isfinite(got.float()).all())
    for part, value in ((got[:, 0, :, ::2], 65504.0), (got[:, 1, :, 1::2], -65504.0)):
        assert bool(((part.double() / value - 1).abs() <= 2.0 ** -11 + 2.0 ** -11).all())     # numerators, the result


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("window", [0, 700])
def test_a_cache_of_nothing_but_infinities_or_nan(value, window):
    """What a model that has diverged leaves in V: prompts, few rows and single tokens over it are right in ordinary time."""
    kv, hd, page, n = 2, 128, 16, 20000
    pages = -(-n // page)
    k = torch.randn(pages, kv, page, hd, device="cuda", dtype=torch.bfloat16)
    v = torch.full_like(k, value)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    for rows in (1, 5, 1500):
        q = torch.randn(rows, 4 * kv * hd, device="cuda", dtype=torch.bfloat16)
        starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        y = ops.paged_attention(ops.PagedCache(k, v), q, table, lens, starts, window=window)
        assert bool(y.isnan().all() if value != value else (y == value).all())
        if rows == 1:
            y = ops.paged_decode(ops.PagedCache(k, v), q, table, lens, window=window)
            assert bool(y.isnan().all() if value != value else (y == value).all())
