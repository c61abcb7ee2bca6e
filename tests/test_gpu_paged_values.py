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


def check(got, layer, planted, window=0, sinks=0, hidden=()):
    """planted: (sequence, position, K / V head, column, value). The columns that hold one are the sum of those that the
    row sees; everything else is the definition's."""
    got = got.cpu()
    want, tol = layer.want(torch.zeros(got.shape), window=window, sinks=sinks, hidden=hidden)
    group, hd = layer.heads // layer.kv, layer.hd
    extra = torch.zeros(got.shape)
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
