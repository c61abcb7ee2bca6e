"""K and V pools that share memory, on a CPU-only host: refused where new rows would be stored, however the strides interleave
them, and nothing else is. Every call here is refused: the ones whose pools are apart, for their input."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from opentars_amd import _lib

P, GB = 0x7F0000000000, 1 << 30
PAGE, HD = 16, 64


def refused_for_pools(shift, kstrides, vstrides, pages, kv, el=2):
    """Whether tars_kv_append refuses these pools (byte strides of page, head, slot; V `shift` bytes behind K) for being one
    memory; otherwise the K rows, which lie in the pool, are what it refuses."""
    pool = _lib.KvPool(P, P + shift, None, None, *kstrides, *vstrides, pages, PAGE, kv, HD, 0 if el == 2 else 2)
    rc = _lib.lib().tars_kv_append(ctypes.byref(pool), P, 0, P + 64 * GB, 0, 0, 1, P + 65 * GB, 0, 4, P + 66 * GB, None, 1, None)
    assert rc == _lib.E_OVERLAP, _lib.last_error()
    return "pools" in _lib.last_error()


def dense(order, n, row, gaps=(0, 0, 0)):
    """Strides of page, head and slot, in `order` from the innermost, each with a gap behind it."""
    s, at = [0, 0, 0], row
    for i, gap in zip(order, gaps):
        s[i] = at + gap
        at = s[i] * n[i]
    return s


def rows_of(base, strides, n, row):
    i, h, t = (np.arange(c) for c in n)
    at = base + (i[:, None, None] * strides[0] + h[None, :, None] * strides[1] + t * strides[2]).reshape(-1)
    return set((at[:, None] + np.arange(0, row, 16)).reshape(-1).tolist())


@pytest.mark.parametrize("el", [1, 2])
def test_pools_that_overlap_are_refused_and_others_are_not(el):
    rng = np.random.default_rng(5)
    row, seen = el * HD, [0, 0]
    for _ in range(1500):
        pages, kv = int(rng.integers(1, 5)), int(rng.integers(1, 4))
        n = (pages, kv, PAGE)
        gaps = [int(rng.choice([0, 0, 16, row, 2 * row])) for _ in range(3)]
        s = dense(rng.permutation(3), n, row, gaps)
        reach = s[0] * pages + s[1] * kv + s[2] * PAGE
        shift = 16 * int(rng.integers(-reach // 16, reach // 16 + 1)) if rng.random() < 0.7 else int(rng.choice([-1, 1])) * int(
            rng.choice([row, *s, s[0] + row, s[2] + row]))
        meet = bool(rows_of(0, s, n, row) & rows_of(shift, s, n, row))
        seen[meet] += 1
        assert refused_for_pools(shift, s, s, pages, kv, el) == meet, (shift, s, n)
    assert min(seen) > 200


def test_pools_of_different_strides():
    """In one block of memory a page: K's part before V's, heads outside slots in one and slots outside heads in the other.
    Where extents of unlike strides meet the pools are refused, whether a row of both does or not."""
    rng = np.random.default_rng(6)
    for _ in range(500):
        pages, kv = int(rng.integers(1, 5)), int(rng.integers(2, 4))
        n, size = (pages, kv, PAGE), 2 * HD * kv * PAGE
        k, v = dense((2, 1, 0), n, 2 * HD), dense((1, 2, 0), n, 2 * HD)
        k[0] = v[0] = 2 * size
        assert not refused_for_pools(size, k, v, pages, kv) and not refused_for_pools(-size, k, v, pages, kv)
        shift = 16 * int(rng.integers(-2 * size // 16, 2 * size // 16))
        if rows_of(0, k, n, 2 * HD) & rows_of(shift, v, n, 2 * HD):
            assert refused_for_pools(shift, k, v, pages, kv)


def test_large_pools():
    n = (1 << 20, 8, PAGE)
    s = dense((2, 1, 0), n, 2 * HD)                                    # 16 KiB a page, 16 GiB
    for shift, meet in ((s[0], True), (-s[0] * (n[0] - 1), True), (s[0] * n[0], False), (-s[0] * n[0], False), (16, True), (s[1], True)):
        assert refused_for_pools(shift, s, s, n[0], n[1]) == meet
    s = [2 * s[0], s[1], s[2]]                                          # K and V page by page
    for shift, meet in ((s[0] // 2, False), (-s[0] // 2, False), (s[0] // 2 - 16, True), (s[0] * 5 + s[0] // 2, False), (s[0] * 5, True)):
        assert refused_for_pools(shift, s, s, n[0], n[1]) == meet
