"""The refusals of the operators around the paged cache (microscaled 4 bits, norm and rotation, log probabilities) at the C ABI, on a
CPU-only host, and what they say of their workspaces. No call here passes validation."""
from __future__ import annotations

import ctypes

import pytest

from opentars_amd import _lib
from test_paged_host import GB, MB, META, P, pool

INF, NAN = float("inf"), float("nan")


def refused(rc):
    assert rc != _lib.OK, "test bug: this call would have launched"
    assert _lib.last_error()
    return rc


# ------------------------------------------------------------------------------------------------ norm and rotation
def rope(store=False, pool_kw=(), **kw):
    a = dict(q=P + 3 * GB, ldq=0, k=P + 4 * GB, ldk=0, v=P + 5 * GB, ldv=0, dtype=0, heads=4, kv_heads=2, hd=128, rows=10,
             qgamma=P + 6 * GB, kgamma=P + 6 * GB + MB, eps=1e-6, tab=P + 7 * GB, positions=100, rot=64, yq=P + 8 * GB, ldyq=0,
             yk=P + 9 * GB, ldyk=0, **META)
    a.update(kw)
    if store:
        p = pool(**dict(pool_kw))
        return refused(_lib.lib().tars_kv_append_rope(
            ctypes.byref(p), a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["dtype"], a["heads"], a["rows"], a["qgamma"],
            a["kgamma"], a["eps"], a["tab"], a["positions"], a["rot"], a["table"], a["ld_table"], a["table_pages"], a["lens"],
            a["starts"], a["seqs"], a["yq"], a["ldyq"], None))
    return refused(_lib.lib().tars_qk_norm_rope(
        a["q"], a["ldq"], a["k"], a["ldk"], a["dtype"], a["heads"], a["kv_heads"], a["hd"], a["rows"], a["qgamma"], a["kgamma"],
        a["eps"], a["tab"], a["positions"], a["rot"], a["lens"], a["starts"], a["seqs"], a["yq"], a["ldyq"], a["yk"], a["ldyk"], None))


BOTH = [
    (dict(q=None), "E_ARG"), (dict(k=None), "E_ARG"), (dict(yq=None), "E_ARG"), (dict(tab=None), "E_ARG"), (dict(lens=None), "E_ARG"),
    (dict(dtype=2), "E_FIELD"), (dict(dtype=-1), "E_FIELD"), (dict(heads=0), "E_FIELD"), (dict(heads=1025), "E_FIELD"),
    (dict(eps=-1e-6), "E_FIELD"), (dict(eps=NAN), "E_FIELD"), (dict(eps=INF), "E_FIELD"), (dict(starts=None), "E_FIELD"),
    (dict(rot=0), "E_ALIGN"), (dict(rot=8), "E_ALIGN"), (dict(rot=24), "E_ALIGN"), (dict(rot=144), "E_ALIGN"), (dict(rot=-16), "E_ALIGN"),
    (dict(positions=0), "E_ALIGN"), (dict(positions=2 ** 30 + 1), "E_RANGE"), (dict(rows=0), "E_ALIGN"), (dict(seqs=0), "E_ALIGN"),
    (dict(rows=2 ** 22 + 1), "E_RANGE"), (dict(seqs=65536, lens=P + 20 * GB, starts=P + 21 * GB), "E_RANGE"),
    (dict(rows=2 ** 22, heads=128, ldq=16 * MB), "E_RANGE"), (dict(tab=P + 7 * GB + 8), "E_ALIGN"), (dict(qgamma=P + 6 * GB + 4), "E_ALIGN"),
    (dict(kgamma=P + 6 * GB + 4), "E_ALIGN"), (dict(lens=P + 2 * GB + 2), "E_ALIGN"), (dict(starts=P + 2 * GB + 2 * MB + 1), "E_ALIGN"),
    (dict(q=P + 3 * GB + 8), "E_ALIGN"), (dict(k=P + 4 * GB + 2), "E_ALIGN"), (dict(yq=P + 8 * GB + 8), "E_ALIGN"),
    (dict(ldq=1008), "E_ALIGN"), (dict(ldq=1032), "E_ALIGN"), (dict(ldk=496), "E_ALIGN"), (dict(ldyq=1000), "E_ALIGN"),
    (dict(ldq=-1024), "E_ALIGN"), (dict(ldq=2 ** 62), "E_RANGE"),
    (dict(yq=P + 3 * GB + 16), "E_OVERLAP"), (dict(yq=P + 3 * GB, ldyq=2048), "E_OVERLAP"),      # not its input as it lies
    (dict(yq=P + 4 * GB + 512), "E_OVERLAP"), (dict(yq=P + 7 * GB + 16), "E_OVERLAP"), (dict(yq=P + 6 * GB), "E_OVERLAP"),
    (dict(yq=P + 2 * GB + MB), "E_OVERLAP"), (dict(yq=P + 2 * GB + 2 * MB - 64), "E_OVERLAP"),
]


@pytest.mark.parametrize("store", [False, True])
@pytest.mark.parametrize("kw,code", BOTH)
def test_rope_refusals(kw, code, store):
    assert rope(store, **kw) == getattr(_lib, code)


@pytest.mark.parametrize("kw,code", [
    (dict(kv_heads=0), "E_FIELD"), (dict(kv_heads=1025), "E_FIELD"), (dict(hd=96), "E_FIELD"), (dict(hd=0), "E_FIELD"),
    (dict(yk=None), "E_ARG"), (dict(yk=P + 9 * GB + 4), "E_ALIGN"), (dict(ldyk=500), "E_ALIGN"), (dict(yk=P + 3 * GB), "E_OVERLAP"),
    (dict(yk=P + 4 * GB + 256), "E_OVERLAP"), (dict(yk=P + 8 * GB + 1024), "E_OVERLAP"), (dict(yk=P + 7 * GB), "E_OVERLAP"),
    (dict(yq=P + 9 * GB, ldyq=2048, yk=P + 9 * GB + 512, ldyk=2048), "E_OVERLAP"),               # columns that share bytes
])
def test_rope_refusals_of_keys(kw, code):
    assert rope(**kw) == getattr(_lib, code)


@pytest.mark.parametrize("kw,code", [
    (dict(v=None), "E_ARG"), (dict(v=P + 5 * GB + 8), "E_ALIGN"), (dict(ldv=500), "E_ALIGN"), (dict(pool_kw=dict(hd=32)), "E_FIELD"),
    (dict(pool_kw=dict(page=48)), "E_FIELD"), (dict(pool_kw=dict(k=None)), "E_ARG"), (dict(table=None), "E_ARG"),
    (dict(pool_kw=dict(v=P)), "E_OVERLAP"), (dict(q=P + 4096), "E_OVERLAP"), (dict(k=P + GB), "E_OVERLAP"), (dict(v=P), "E_OVERLAP"),
    (dict(yq=P + 4096), "E_OVERLAP"), (dict(yq=P + 5 * GB), "E_OVERLAP"), (dict(tab=P + GB + 512), "E_OVERLAP"),
    (dict(qgamma=P + 64), "E_OVERLAP"),
])
def test_rope_refusals_of_the_pool(kw, code):
    assert rope(True, **kw) == getattr(_lib, code)


# ------------------------------------------------------------------------------------------------ microscaled 4 bits
def mx(at, n, width, **kw):
    a = dict(values=P + at, scales=P + at + GB, ld_values=0, ld_scales=0, rows=n, k=width)
    a.update(kw)
    return _lib.Mx4(*(a[f] for f, _ in _lib.Mx4._fields_))


BAD_MX = [
    (dict(values=None), "E_ARG"), (dict(scales=None), "E_ARG"), (dict(rows=0), "E_ALIGN"), (dict(rows=-1), "E_ALIGN"),
    (dict(k=0), "E_ALIGN"), (dict(k=48), "E_ALIGN"), (dict(ld_values=240), "E_ALIGN"), (dict(ld_values=264), "E_ALIGN"),
    (dict(ld_scales=8), "E_ALIGN"), (dict(ld_scales=24), "E_ALIGN"), (dict(values=P + 8), "E_ALIGN"), (dict(scales=P + GB + 4), "E_ALIGN"),
    (dict(ld_values=-512), "E_ALIGN"), (dict(k=2 ** 20 + 32), "E_RANGE"), (dict(ld_values=2 ** 22 + 16), "E_RANGE"),
    (dict(ld_scales=2 ** 22 + 16), "E_RANGE"), (dict(rows=2 ** 24 + 1), "E_RANGE"),
]


def quant(dst_kw=(), **kw):
    a = dict(x=P + 8 * GB, ldx=0, dtype=1)
    a.update(kw)
    m = mx(0, 10, 512, **dict(dst_kw))
    return refused(_lib.lib().tars_quant_mx4(a["x"], a["ldx"], a["dtype"], None if a.get("none") else ctypes.byref(m), None))


@pytest.mark.parametrize("kw,code", [(dict(dst_kw=k), c) for k, c in BAD_MX] + [
    (dict(x=None), "E_ARG"), (dict(none=True), "E_ARG"), (dict(dtype=2), "E_FIELD"), (dict(dtype=4), "E_FIELD"),
    (dict(x=P + 8 * GB + 8), "E_ALIGN"), (dict(ldx=1016), "E_ALIGN"), (dict(ldx=1000), "E_ALIGN"), (dict(x=P), "E_OVERLAP"),
    (dict(x=P + GB + 64), "E_OVERLAP"), (dict(dst_kw=dict(scales=P + 256)), "E_OVERLAP"),
])
def test_quant_refusals(kw, code):
    assert quant(**kw) == getattr(_lib, code)


def product(x_kw=(), w_kw=(), quantises=False, **kw):
    a = dict(x=P + 8 * GB, ldx=0, dtype=1, M=10, bias=P + 6 * GB, y=P + 7 * GB, ldy=0, out=1, work=P + 12 * GB, work_bytes=GB)
    a.update(kw)
    x, w = mx(3 * GB, 10, 512, **dict(x_kw)), mx(0, 100, 512, **dict(w_kw))
    rest = ctypes.byref(w), a["bias"], a["y"], a["ldy"], a["out"], a["work"], a["work_bytes"], None
    if quantises:
        return refused(_lib.lib().tars_quant_gemm_mx4(a["x"], a["ldx"], a["dtype"], a["M"], *rest))
    return refused(_lib.lib().tars_gemm_mx4(ctypes.byref(x), *rest))


@pytest.mark.parametrize("quantises", [False, True])
@pytest.mark.parametrize("kw,code", [(dict(w_kw=k), c) for k, c in BAD_MX] + [
    (dict(y=None), "E_ARG"), (dict(out=2), "E_FIELD"), (dict(out=-1), "E_FIELD"), (dict(y=P + 7 * GB + 1), "E_ALIGN"),
    (dict(ldy=198), "E_ALIGN"), (dict(ldy=201), "E_ALIGN"), (dict(bias=P + 6 * GB + 2), "E_ALIGN"), (dict(ldy=-400), "E_ALIGN"),
    (dict(ldy=2 ** 62), "E_RANGE"), (dict(y=P), "E_OVERLAP"), (dict(y=P + GB + 16), "E_OVERLAP"), (dict(y=P + 6 * GB + 200), "E_OVERLAP"),
])
def test_product_refusals(kw, code, quantises):
    assert product(quantises=quantises, **kw) == getattr(_lib, code)


def test_product_refusals_of_x():
    for kw, code in BAD_MX:
        at = {f: v + 3 * GB if f in ("values", "scales") and v else v for f, v in kw.items()}
        assert product(x_kw=at) == getattr(_lib, code)
    assert product(x_kw=dict(k=544)) == _lib.E_FIELD                   # the two disagree on k
    assert product(x_kw=dict(rows=2 ** 22 + 1)) == _lib.E_RANGE
    assert product(x_kw=dict(rows=2 ** 22), w_kw=dict(rows=2 ** 17)) == _lib.E_RANGE
    assert product(y=P + 3 * GB + 64) == _lib.E_OVERLAP and product(y=P + 4 * GB) == _lib.E_OVERLAP


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), "E_ARG"), (dict(dtype=2), "E_FIELD"), (dict(dtype=5), "E_FIELD"), (dict(M=0), "E_ALIGN"), (dict(M=2 ** 22 + 1), "E_RANGE"),
    (dict(x=P + 8 * GB + 4), "E_ALIGN"), (dict(ldx=1000), "E_ALIGN"), (dict(ldx=1032), "E_ALIGN"), (dict(x=P + 7 * GB + 64), "E_OVERLAP"),
    (dict(M=2 ** 22, w_kw=dict(rows=2 ** 17)), "E_RANGE"),
])
def test_product_refusals_of_rows(kw, code):
    assert product(quantises=True, **kw) == getattr(_lib, code)


@pytest.mark.parametrize("quantises", [False, True])
@pytest.mark.parametrize("M,N,K", [(100, 1024, 8192), (112, 11, 4352), (300, 64, 65536), (5000, 100, 512), (64, 64, 4096)])
def test_product_workspaces(M, N, K, quantises):
    need = _lib.lib().tars_mx4_workspace(M, N, K, quantises)
    assert 0 <= need < GB
    codes = M * (K // 2 + 16 * -(-K // 512)) if quantises else 0
    assert need >= codes
    if need:
        kw = dict(quantises=quantises, x_kw=dict(rows=M, k=K), w_kw=dict(rows=N, k=K), M=M)
        assert product(work_bytes=need - 1, **kw) == _lib.E_RANGE
        assert product(work=None, **kw) == _lib.E_ARG
        assert product(work=P + 12 * GB + 8, **kw) == _lib.E_ALIGN
        for at in (0, GB, 6 * GB, 7 * GB, 8 * GB if quantises else 3 * GB):
            assert product(work=P + at + 16 - need // 16 * 16, **kw) == _lib.E_OVERLAP


def test_no_workspace_for_products_that_are_refused():
    ws = _lib.lib().tars_mx4_workspace
    assert ws(100, 1024, 8192, 0) > 0 and ws(100, 1024, 8192, 1) > 0
    for q in (0, 1):
        for bad in ((0, 1024, 8192), (-5, 1024, 8192), (100, 0, 8192), (100, 1024, 0), (100, 1024, 8208), (100, 1024, 2 ** 20 + 32),
                    (2 ** 22 + 1, 1, 512), (100, 2 ** 24 + 1, 512), (2 ** 22, 2 ** 17, 512), (100, 1024, -32)):
            assert ws(*bad, q) == 0, bad


# ------------------------------------------------------------------------------------------------ log probabilities
def logprobs(**kw):
    a = dict(x=P, ld=0, dtype=1, rows=3, vocab=1000, tokens=P + GB, ld_tokens=0, wide=0, given=2, lp=P + 2 * GB, h=P + 3 * GB, top=5,
             tv=P + 4 * GB, ti=P + 5 * GB, work=P + 6 * GB, work_bytes=GB)
    a.update(kw)
    return refused(_lib.lib().tars_token_logprobs(a["x"], a["ld"], a["dtype"], a["rows"], a["vocab"], a["tokens"], a["ld_tokens"], a["wide"],
                                                  a["given"], a["lp"], a["h"], a["top"], a["tv"], a["ti"], a["work"], a["work_bytes"], None))


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), "E_ARG"), (dict(h=None), "E_ARG"), (dict(tokens=None), "E_ARG"), (dict(lp=None), "E_ARG"), (dict(tv=None), "E_ARG"),
    (dict(ti=None), "E_ARG"), (dict(dtype=2), "E_FIELD"), (dict(dtype=9), "E_FIELD"), (dict(wide=2), "E_FIELD"), (dict(given=-1), "E_FIELD"),
    (dict(given=65537), "E_FIELD"), (dict(top=-1), "E_FIELD"), (dict(top=65), "E_FIELD"), (dict(top=5, vocab=4), "E_FIELD"),
    (dict(rows=0), "E_ALIGN"), (dict(vocab=0, top=0), "E_ALIGN"), (dict(rows=2 ** 22 + 1), "E_RANGE"), (dict(vocab=2 ** 24 + 1), "E_RANGE"),
    (dict(ld=1998), "E_ALIGN"), (dict(ld=2001), "E_ALIGN"), (dict(ld=-2000), "E_ALIGN"), (dict(ld_tokens=4), "E_ALIGN"),
    (dict(ld_tokens=10), "E_ALIGN"), (dict(wide=1, ld_tokens=20), "E_ALIGN"), (dict(wide=1, tokens=P + GB + 4), "E_ALIGN"),
    (dict(x=P + 1), "E_ALIGN"), (dict(dtype=0, x=P + 2), "E_ALIGN"), (dict(lp=P + 2 * GB + 2), "E_ALIGN"), (dict(h=P + 3 * GB + 1), "E_ALIGN"),
    (dict(tv=P + 4 * GB + 2), "E_ALIGN"), (dict(ti=P + 5 * GB + 3), "E_ALIGN"), (dict(ld=2 ** 62, rows=5), "E_RANGE"),
    (dict(ld_tokens=2 ** 62, rows=5), "E_RANGE"), (dict(h=P + 1000), "E_OVERLAP"), (dict(lp=P), "E_OVERLAP"), (dict(tv=P + GB), "E_OVERLAP"),
    (dict(ti=P + 4 * GB + 16), "E_OVERLAP"), (dict(h=P + 2 * GB + 8), "E_OVERLAP"), (dict(ti=P + 3 * GB), "E_OVERLAP"),
])
def test_logprobs_refusals(kw, code):
    assert logprobs(**kw) == getattr(_lib, code)


@pytest.mark.parametrize("rows,vocab,top", [(1, 152064, 5), (1, 200000, 64), (8, 50000, 0), (64, 152064, 1)])
def test_logprobs_workspaces(rows, vocab, top):
    need = _lib.lib().tars_logprobs_workspace(rows, vocab, 1, top)
    assert 0 <= need < GB and (need > 0 or rows == 8)                  # short rows are not parted
    if need == 0:
        return
    kw = dict(rows=rows, vocab=vocab, top=top)
    assert logprobs(work_bytes=need - 1, **kw) == _lib.E_RANGE and logprobs(work=None, **kw) == _lib.E_ARG
    assert logprobs(work=P + 6 * GB + 8, **kw) == _lib.E_ALIGN
    for at in (0, GB, 2 * GB, 3 * GB):
        assert logprobs(work=P + at, **kw) == _lib.E_OVERLAP


def test_no_workspace_for_log_probabilities_that_are_refused():
    ws = _lib.lib().tars_logprobs_workspace
    for bad in ((0, 152064, 1, 5), (-1, 152064, 1, 5), (1, 0, 1, 0), (1, 152064, 2, 5), (1, 152064, 7, 5), (1, 152064, 1, 65),
                (1, 152064, 1, -1), (2 ** 22 + 1, 152064, 1, 5), (1, 2 ** 24 + 1, 1, 5)):
        assert ws(*bad) == 0, bad
