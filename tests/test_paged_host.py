"""The paged key / value cache on a CPU-only host: its index arithmetic (compiled as plain C++) against walks over the
positions, and the C ABI's refusals. No call here passes validation."""
from __future__ import annotations

import ctypes
import subprocess

import numpy as np
import pytest

from opentars_amd import _lib, build

P, MB, GB = 0x7F0000000000, 1 << 20, 1 << 30
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "index.cpp").write_text(r'''
#include <cstdio>
#include "paged_index.h"
using namespace tars;
int main() {
  char what;
  int v[6];
  while (std::scanf(" %c", &what) == 1) {
    for (int& x : v) if (std::scanf("%d", &x) != 1) return 1;
    if (what == 's') {
      const Steps s = visible_steps(v[0], v[1], v[2], v[3], v[4], v[5]);
      std::printf("%d %d %d\n", s.a, s.b0, s.b1);
    } else if (what == 'r') {
      const int32_t starts[2] = {v[0], v[1]};
      const RowSpan r = seq_rows(starts, 0, v[2]);
      std::printf("%d %d 0\n", r.first, r.n);
    } else if (what == 'l') {
      const int32_t len = v[0];
      std::printf("%d 0 0\n", seq_len(&len, 0, v[1]));
    } else if (what == 't') {
      const int32_t starts[2] = {v[0], v[1]};
      std::printf("%d %d 0\n", tile_first(starts, 0, v[2], v[3], v[4]), tile_first(starts, 1, v[2], v[3], v[4]));
    } else if (what == 'b') {
      std::printf("%d 0 0\n", tiles_behind(v[0], v[1], v[2], v[3], v[4], v[5]));
    } else {
      std::printf("%d 0 0\n", sees(v[0], v[1], v[2], v[3]));
    }
  }
}
''')
    exe = d / "index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-Wall", "-Werror",
                    "-I", str(build.CSRC), str(d / "index.cpp"), "-o", str(exe)], check=True, capture_output=True)

    def ask(lines):
        out = subprocess.run([str(exe)], input="\n".join("%s %d %d %d %d %d %d" % (*l, *[0] * (7 - len(l))) for l in lines),
                             capture_output=True, text=True, check=True).stdout
        return np.array([int(x) for x in out.split()]).reshape(-1, 3)
    return ask


def test_visible_steps_hold_every_seen_position_once(index):
    rng = np.random.default_rng(0)
    cases = []
    for _ in range(4000):
        n = int(rng.integers(0, 300))
        r = int(rng.integers(1, 80))
        plo = n - r if rng.random() < 0.7 else int(rng.integers(-50, n + 1)) - 1      # rows are at positions below n
        cases.append((plo, min(n - 1, plo + int(rng.integers(0, r))), n, int(rng.choice([0, 1, 5, 16, 33, 100, 400, TOP])),
                      int(rng.choice([0, 1, 4, 16, 40, 90, TOP])), int(rng.choice([16, 32, 64]))))
    for (plo, phi, n, w, s, step), (a, b0, b1) in zip(cases, index([("s", *c) for c in cases])):
        assert 0 <= a <= b0 <= b1 <= (max(n, 0) + step - 1) // step
        steps = list(range(a)) + list(range(b0, b1))
        held = {j for t in steps for j in range(t * step, t * step + step)}
        seen = {j for p in range(plo, phi + 1) for j in range(min(n, p + 1)) if w == 0 or j > p - w or j < s}
        assert seen <= held, (plo, phi, n, w, s, step)
        for t in steps:                                                # and no step is wholly unseen
            assert seen & set(range(t * step, t * step + step)), (plo, phi, n, w, s, step, t)


def test_visible_steps_at_the_ends_of_32_bits(index):
    top = 2 ** 30
    cases = [(top - 1, top - 1, top, w, s, 64) for w in (0, 1, 512, TOP) for s in (0, 4, TOP)]
    cases += [(-2 ** 22, -1, top, TOP, TOP, 16), (-2 ** 22, top - 1, top, TOP, 0, 16)]
    for (plo, phi, n, w, s, step), (a, b0, b1) in zip(cases, index([("s", *c) for c in cases])):
        assert 0 <= a <= b0 <= b1 <= n // step
        if phi < 0:
            assert a + b1 - b0 == 0
        elif w in (0, TOP):
            assert a + b1 - b0 == n // step
        else:
            assert b1 == n // step and b0 == max((n - w) // step, a) and a == min(-(-min(s, n - w) // step), b1)


def test_sees_rows_and_lengths(index):
    rng = np.random.default_rng(1)
    q = [(int(p), int(j), int(w), int(s)) for p, j, w, s in zip(rng.integers(0, 60, 2000), rng.integers(0, 60, 2000),
                                                               rng.integers(0, 30, 2000), rng.integers(0, 30, 2000))]
    q += [(2 ** 30, 2 ** 30, TOP, TOP), (0, 0, TOP, 0), (5, 0, 5, 0)]
    got = index([("v", *c) for c in q])[:, 0]
    assert got.tolist() == [int(j <= p and (w == 0 or j > p - w or j < s)) for p, j, w, s in q]
    bad = [-2 ** 31, -1, 0, 3, 7, 8, 9, TOP]
    rows = [(a, b, 8) for a in bad for b in bad]
    for (a, b, n), (first, count, _) in zip(rows, index([("r", *r) for r in rows])):
        lo, hi = min(max(a, 0), n), min(max(b, 0), n)
        assert (first, count) == (lo, max(hi - lo, 0)) and first + count <= n
    assert index([("l", v, 8) for v in bad])[:, 0].tolist() == [min(max(v, 0), 8) for v in bad]


def test_every_sequence_has_numbers_for_its_tiles(index):
    rng = np.random.default_rng(2)
    rows = 1 << 18
    cases = [(int(a), int(a + n), rows, int(g), 128) for a, n, g in
             zip(rng.integers(0, rows // 2, 3000), rng.integers(0, 600, 3000), rng.integers(1, 1025, 3000))]
    cases += [(0, 1 << 22, 1 << 22, 64, 128), ((1 << 22) - 1, 1 << 22, 1 << 22, 64, 128), (0, 0, 1, 1024, 128)]
    for (a, b, _, g, m), (first, after, _) in zip(cases, index([("t", *c) for c in cases])):
        assert first == a * g // m                                     # of sequence 0: no numbers lost before it
        assert -(-(b - a) * g // m) <= after - first <= -(-(b - a) * g // m) + 1
    # numbers past the last tile are few: one for each sequence
    assert index([("t", -5, 2 ** 31 - 1, 100, 3, 128)])[0].tolist() == [0, 300 // 128 + 1, 0]


def test_tiles_behind_a_step(index):
    rng = np.random.default_rng(3)
    cases = [(int(s), int(p0), int(n), int(g), int(m), int(step)) for s, p0, n, g, m, step in
             zip(rng.integers(-1, 20, 4000), rng.integers(-70, 300, 4000), rng.integers(0, 300, 4000),
                 rng.choice([1, 2, 3, 8, 40, 200], 4000), rng.choice([16, 128], 4000), rng.choice([32, 64], 4000))]
    for (s, p0, n, g, m, step), (got, _, _) in zip(cases, index([("b", *c) for c in cases])):
        last = [min(((t + 1) * m - 1) // g, n - 1) for t in range(-(-n * g // m))]
        assert got == (len(last) if s <= 0 else sum(p0 + x >= (s - 1) * step for x in last)), (s, p0, n, g, m, step)
    top = 2 ** 30                                                       # the longest cache, the most rows
    assert index([("b", top // 64, top - 2 ** 22, 2 ** 22, 64, 128, 64), ("b", top // 64 + 2, top - 2 ** 22, 2 ** 22, 64, 128, 64),
                  ("b", 1, top - 2 ** 22, 2 ** 22, 64, 128, 64)])[:, 0].tolist() == [32, 0, 2 ** 21]


def pool(**kw):
    page, hd, kv, pages, el = kw.get("page", 16), kw.get("hd", 128), kw.get("kv_heads", 2), kw.get("pages", 8), 2
    slot, head = el * hd, el * hd * page
    a = dict(k=P, v=P + GB, kscale=None, vscale=None, k_page=head * kv, k_head=head, k_slot=slot, v_page=head * kv,
             v_head=head, v_slot=slot, pages=pages, page=page, kv_heads=kv, hd=hd, dtype=0)
    a.update(kw)
    return _lib.KvPool(*(a[f] for f, _ in _lib.KvPool._fields_))


META = dict(table=P + 2 * GB, ld_table=0, table_pages=4, lens=P + 2 * GB + MB, starts=P + 2 * GB + 2 * MB, seqs=3)


def append(pool_kw=(), **kw):
    a = dict(k=P + 3 * GB, ldk=0, v=P + 3 * GB + MB, ldv=0, dtype=0, rows=10, **META)
    a.update(kw)
    p = pool(**dict(pool_kw))
    rc = _lib.lib().tars_kv_append(None if a.get("no_pool") else ctypes.byref(p), a["k"], a["ldk"], a["v"], a["ldv"], a["dtype"],
                                   a["rows"], a["table"], a["ld_table"], a["table_pages"], a["lens"], a["starts"], a["seqs"],
                                   None)
    assert rc != _lib.OK, "test bug: this call would have launched"
    return rc


def attend(pool_kw=(), decode=False, **kw):
    a = dict(q=P + 3 * GB, ldq=0, dtype=0, heads=4, rows=10, y=P + 4 * GB, ldy=0, out=1, scale=0.1, window=0, sinks=0,
             work=P + 5 * GB, work_bytes=GB, **META)
    a.update(kw)
    p = pool(**dict(pool_kw))
    head = (ctypes.byref(p), a["q"], a["ldq"], a["dtype"], a["heads"], a["seqs"] if decode else a["rows"], a["y"], a["ldy"],
            a["out"], a["scale"], a["window"], a["sinks"], a["table"], a["ld_table"], a["table_pages"], a["lens"])
    if decode:
        rc = _lib.lib().tars_paged_decode(*head, a["work"], a["work_bytes"], None)
    else:
        rc = _lib.lib().tars_paged_attention(*head, a["starts"], a["seqs"], a["work"], a["work_bytes"], None)
    assert rc != _lib.OK, "test bug: this call would have launched"
    return rc


SHARED = [
    (dict(pool_kw=dict(k=None)), "E_ARG"), (dict(table=None), "E_ARG"), (dict(lens=None), "E_ARG"),
    (dict(dtype=2), "E_FIELD"), (dict(dtype=1), "E_FIELD"), (dict(pool_kw=dict(dtype=3)), "E_FIELD"),
    (dict(pool_kw=dict(kscale=P + 9 * GB)), "E_FIELD"),                # scales of a pool that is not E4M3
    (dict(pool_kw=dict(hd=96)), "E_FIELD"), (dict(pool_kw=dict(hd=32)), "E_FIELD"),
    (dict(pool_kw=dict(page=8)), "E_FIELD"), (dict(pool_kw=dict(page=48)), "E_FIELD"),
    (dict(pool_kw=dict(kv_heads=0)), "E_FIELD"), (dict(pool_kw=dict(kv_heads=1025)), "E_FIELD"),
    (dict(pool_kw=dict(pages=0)), "E_ALIGN"), (dict(table_pages=0), "E_ALIGN"), (dict(ld_table=12), "E_ALIGN"),
    (dict(ld_table=18), "E_ALIGN"), (dict(table=P + 2 * GB + 2), "E_ALIGN"), (dict(lens=P + 2), "E_ALIGN"),
    (dict(pool_kw=dict(k=P + 8)), "E_ALIGN"), (dict(pool_kw=dict(k_slot=264)), "E_ALIGN"),
    (dict(pool_kw=dict(k_slot=128)), "E_ALIGN"),                       # slots that share bytes
    (dict(pool_kw=dict(v_page=0)), "E_ALIGN"), (dict(pool_kw=dict(v_head=-4096)), "E_ALIGN"),
    (dict(pool_kw=dict(k_page=2 ** 62, pages=100)), "E_ALIGN"),        # an extent past the address space
    (dict(table_pages=2 ** 26, pool_kw=dict(page=32)), "E_RANGE"),
    (dict(pool_kw=dict(k_slot=2 ** 26 + 16, k_head=2 ** 32, k_page=2 ** 34)), "E_RANGE"),
]


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(no_pool=True), "E_ARG"), (dict(k=None), "E_ARG"), (dict(rows=0), "E_ALIGN"), (dict(seqs=0), "E_ALIGN"),
    (dict(starts=None), "E_FIELD"), (dict(rows=2 ** 22 + 1), "E_RANGE"), (dict(starts=P + 2 * GB + 2 * MB + 1), "E_ALIGN"),
    (dict(ldk=256), "E_ALIGN"), (dict(ldv=520), "E_ALIGN"), (dict(v=P + 3 * GB + 8), "E_ALIGN"),
    (dict(pool_kw=dict(v=P)), "E_OVERLAP"), (dict(k=P + 4096), "E_OVERLAP"), (dict(lens=P + GB + 64), "E_OVERLAP"),
])
def test_append_refusals(kw, code):
    assert append(**kw) == getattr(_lib, code)
    assert _lib.last_error()


@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(q=None), "E_ARG"), (dict(y=None), "E_ARG"), (dict(heads=3), "E_FIELD"), (dict(heads=0), "E_FIELD"),
    (dict(heads=1026), "E_FIELD"), (dict(out=2), "E_FIELD"), (dict(out=3), "E_FIELD"), (dict(scale=0.0), "E_FIELD"),
    (dict(scale=-1.0), "E_FIELD"), (dict(scale=float("inf")), "E_FIELD"), (dict(scale=float("nan")), "E_FIELD"),
    (dict(window=-1), "E_FIELD"), (dict(sinks=-2), "E_FIELD"), (dict(ldq=1016), "E_ALIGN"), (dict(ldy=1000), "E_ALIGN"),
    (dict(y=P + 4 * GB + 4), "E_ALIGN"), (dict(y=P + 3 * GB + 1008), "E_OVERLAP"), (dict(y=P + GB), "E_OVERLAP"),
    (dict(y=P + 2 * GB - 64), "E_OVERLAP"),
])
def test_attention_refusals(kw, code, decode):
    assert attend(decode=decode, **kw) == getattr(_lib, code)
    assert _lib.last_error()


def test_counts_past_the_launch_limits():
    far = dict(lens=P + 6 * GB, starts=P + 7 * GB, table_pages=1)
    assert append(seqs=65536, **far) == attend(seqs=65536, **far) == attend(decode=True, seqs=65536, **far) == _lib.E_RANGE
    kw = dict(pool_kw=dict(kv_heads=1), heads=1024, seqs=4097, **far)
    assert attend(**kw) == attend(decode=True, **kw) == _lib.E_RANGE
    assert attend(pool_kw=dict(kv_heads=1), heads=128, rows=2 ** 21 + 1) == _lib.E_RANGE


def test_attention_needs_starts():
    assert attend(starts=None) == _lib.E_ARG
    assert attend(rows=0) == _lib.E_ALIGN and attend(decode=True, seqs=0) == _lib.E_ALIGN


def test_workspace():
    ws = _lib.lib().tars_paged_workspace
    for decode in (0, 1):
        for heads, kv, hd, rows, seqs, width, page in ((32, 8, 128, 3, 3, 4096, 64), (16, 8, 128, 1, 1, 2 ** 20, 1024),
                                                       (4, 1, 256, 100, 100, 512, 16), (1024, 1, 64, 1, 1, 64, 16)):
            need = ws(heads, kv, hd, rows, seqs, width, page, decode)
            assert 0 <= need < 1 << 30
            if need:
                kw = dict(pool_kw=dict(kv_heads=kv, hd=hd, page=page), heads=heads, rows=rows, seqs=seqs, table_pages=width,
                          lens=P + 6 * GB, starts=P + 7 * GB)
                assert attend(decode=bool(decode), work_bytes=need - 1, **kw) == _lib.E_RANGE
                assert attend(decode=bool(decode), work=None, **kw) == _lib.E_ARG
                assert attend(decode=bool(decode), work=P + 5 * GB + 4, **kw) == _lib.E_ALIGN
                assert attend(decode=bool(decode), work=P + 64, **kw) == _lib.E_OVERLAP
        assert ws(3, 2, 128, 1, 1, 4, 16, decode) == 0 and ws(4, 2, 128, 1, 0, 4, 16, decode) == 0
        assert ws(4, 2, 128, 1, 1, 2 ** 30, 16, decode) == 0
