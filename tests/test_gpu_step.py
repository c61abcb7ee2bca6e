"""A serving step's operators together on the GPU, as a program runs them: products in microscaled 4 bits around queries and keys
that are normed, rotated and stored, attention over the pages, and the log probabilities of the head's logits. Each step is
held against its definition in 64 bits, of what the step before it gave. Needs a gfx950 GPU."""
from __future__ import annotations

import math

import pytest
import torch

from opentars_amd import ops
from opentars_amd.contract import OUT_FP32
from paged_data import Layer, bits, compare
from step_data import HALF, TINY, logprobs, packed, quantised, random_codes, rotated, table, values_of

pytestmark = pytest.mark.gpu
HEADS, KV, HD, DIM, VOCAB = 4, 2, 128, 512, 1009
LENS, ROWS = [40, 1, 17, 100], [33, 1, 1, 20]


def on_gpu(w):
    return ops.Mx4(packed(w[0]).cuda(), w[1].to(torch.uint8).cuda())


class Model:
    """One layer and a head; `rows` new rows of sequences of LENS positions, whose older keys and values are in the pool."""

    def __init__(self, rows, qt):
        g = torch.Generator().manual_seed(sum(rows))
        self.layer = Layer(3, LENS, rows, HEADS, KV, HD, qt=qt)
        self.decode = rows == [1] * len(rows)
        shapes = [((HEADS + 2 * KV) * HD, DIM), (DIM, HEADS * HD), (VOCAB, DIM)]
        self.w = [random_codes(g, *s, low=122, spread=3) for s in shapes]
        self.wd = [on_gpu(w) for w in self.w]
        self.bias = 0.1 * torch.randn(shapes[0][0], generator=g)
        self.gamma = 1 + 0.2 * torch.randn(2, HD, generator=g)
        self.tab = table(128, HD)
        self.h = torch.randn(3, sum(rows), DIM, generator=g).to(self.layer.qt)
        self.tokens = torch.randint(0, VOCAB, (len(rows), 2), generator=g)
        self.cache, _, self.table, self.lens, self.starts = self.layer.dev(ops)
        self.consts = self.bias.cuda(), self.gamma.cuda(), self.tab.cuda(), self.tokens.cuda()
        self.last = torch.tensor([sum(rows[:b + 1]) - 1 for b in range(len(rows))]).cuda()

    def step(self, h):
        bias, gamma, tab, tokens = self.consts
        starts = None if self.decode else self.starts
        qkv = ops.gemm_mx4(h, self.wd[0], bias)
        q, k, v = qkv.split([HEADS * HD, KV * HD, KV * HD], 1)
        yq = ops.kv_append_rope(self.cache, q, k, v, self.table, self.lens, tab, starts, gamma[0], gamma[1])
        if self.decode:
            att = ops.paged_decode(self.cache, yq, self.table, self.lens)
        else:
            att = ops.paged_attention(self.cache, yq, self.table, self.lens, self.starts)
        y = ops.gemm_mx4(att, self.wd[1])
        last = y.index_select(0, self.last)
        logits = ops.gemm_mx4(last, self.wd[2], out=OUT_FP32)
        return qkv, yq, att, y, last, logits, ops.token_logprobs(logits, tokens, top=5)


def check_product(got, x, w, bias=None):
    a, b = values_of(*quantised(x.cpu())), values_of(*w)
    want, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.abs().double()
    tol = (8 + 2 * math.sqrt(x.shape[1])) * 2.0 ** -24 * size
    tol += HALF[got.dtype] * (want.abs() + tol) + TINY[got.dtype]
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("qt", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [ROWS, [1] * 4], ids=["prompts", "tokens"])
def test_each_step_of_a_run(rows, qt):
    m = Model(rows, qt)
    layer = m.layer
    qkv, yq, att, y, last, logits, r = m.step(m.h[0].cuda())
    check_product(qkv, m.h[0], m.w[0], m.bias)
    at = [(sum(rows[:b]) + i, n - c + i) for b, (n, c) in enumerate(zip(LENS, rows)) for i in range(c)]
    p = torch.tensor([pos for _, pos in at])
    for got, x, gamma in ((yq, qkv[:, :HEADS * HD], m.gamma[0]),
                          (None, qkv[:, HEADS * HD:(HEADS + KV) * HD], m.gamma[1])):
        want, tol = rotated(x.cpu(), gamma, m.tab, p, HD, 1e-6)
        tol = tol + HALF[layer.qt] * (want.abs() + tol) + TINY[layer.qt]
        if got is None:
            where = [layer.where[b][n - c + i] for b, (n, c) in enumerate(zip(LENS, rows)) for i in range(c)]
            pool = m.cache.k.cpu()
            got = torch.stack([pool[pg, :, slot] for pg, slot in where])
        assert ((got.cpu().double().view(want.shape) - want).abs() <= tol).all()
    # the attention of what the pages hold now
    k, v = m.cache.k.cpu().double(), m.cache.v.cpu().double()
    layer.K = [torch.stack([k[pg, :, slot] for pg, slot in w]) for w in layer.where]
    layer.V = [torch.stack([v[pg, :, slot] for pg, slot in w]) for w in layer.where]
    assert torch.equal(layer.V[0][-1].flatten(), qkv[sum(rows[:1]) - 1, (HEADS + KV) * HD:].cpu().double())
    layer.q = yq.cpu()
    want, tol = layer.want(torch.zeros(att.shape, dtype=layer.qt))
    compare(att, want, tol)
    check_product(y, att, m.w[1])
    check_product(logits, last, m.w[2])
    for i in range(len(rows)):
        given, h, tv, ti = logprobs(logits[i].cpu(), m.tokens[i].tolist(), 5)
        x = logits[i].double()
        tol = (16 + 2 * math.sqrt(VOCAB)) * 2.0 ** -24 + 8 * 2.0 ** -24 * max(20.0, float(x.max() - x.min()))
        assert r.top_ids[i].tolist() == ti
        for got, w in ((r.logprobs[i], given), (r.entropy[i:i + 1], [h]), (r.top_logprobs[i], tv)):
            assert ((got.cpu().double() - torch.tensor(w, dtype=torch.float64)).abs() <= tol).all()


@pytest.mark.parametrize("rows", [ROWS, [1] * 4], ids=["prompts", "tokens"])
def test_a_captured_run_replayed(rows):
    """The whole step in a graph, replayed with other rows between eager steps of the same model into another cache."""
    m, other = Model(rows, "bf16"), Model(rows, "bf16")
    hs = [h.cuda() for h in m.h]
    flat = lambda out: [*out[:6], *out[6]]  # noqa: E731
    eager = []
    for h in hs:
        eager.append([t.clone() for t in flat(other.step(h))] + [other.cache.k.clone(), other.cache.v.clone()])
    buf = hs[0].clone()
    m.step(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(buf)
    for i in (1, 0, 2, 2, 1):
        buf.copy_(hs[i])
        torch.cuda.synchronize()
        graph.replay()
        other.step(hs[(i + 1) % 3])
        torch.cuda.synchronize()
        for got, want in zip([*flat(out), m.cache.k, m.cache.v], eager[i]):
            kind = torch.int32 if got.element_size() == 4 else torch.int16
            assert torch.equal(got.contiguous().view(kind), want.contiguous().view(kind))


def test_a_queue_of_products_of_one_quantised_input():
    """An input quantised once serves several weights, and gives what each call gives by itself."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(70, 512, generator=g).bfloat16().cuda()
    q = ops.quant_mx4(x)
    for n in (64, 300, 1000):
        w = on_gpu(random_codes(g, n, 512, low=120, spread=4))
        assert torch.equal(bits(ops.gemm_mx4(q, w).cpu()), bits(ops.gemm_mx4(x, w).cpu()))


# ------------------------------------------------------------------------------------------------ the ends of the ranges
@pytest.mark.parametrize("M,N,K", [(1, 16, 2 ** 20), (50, 3, 2 ** 20), (1, 300001, 32), (70001, 3, 64), (49, 70000, 32), (200, 24, 2 ** 18)])
def test_products_at_the_ends(M, N, K):
    g = torch.Generator().manual_seed(M + N)
    x, w = random_codes(g, M, K, low=124, spread=4), random_codes(g, N, K, low=124, spread=4)
    a, b = values_of(*x), values_of(*w)
    want, size = a @ b.T, a.abs() @ b.abs().T
    got = ops.gemm_mx4(on_gpu(x), on_gpu(w), out=OUT_FP32)
    tol = (8 + 2 * math.sqrt(K)) * 2.0 ** -24 * size
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("rows,vocab,top,dt", [(1, 2 ** 24, 64, torch.float32), (70001, 3, 3, torch.bfloat16), (1, 2 ** 24, 0, torch.bfloat16),
                                               (257, 20000, 7, torch.float16), (70, 262144, 64, torch.bfloat16)])
def test_log_probabilities_at_the_ends(rows, vocab, top, dt):
    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(dt)
    t = torch.randint(-1, vocab, (rows, 2), generator=g)
    r = ops.token_logprobs(x.cuda(), t.cuda(), top=top)
    for i in {0, 1, rows // 2, rows - 2, rows - 1} & set(range(rows)):
        d = x[i].double()
        lp = torch.log_softmax(d, 0)
        tol = (16 + 2 * math.sqrt(vocab)) * 2.0 ** -24 + 8 * 2.0 ** -24 * max(20.0, float(d.max() - d.min()))
        order = torch.sort(d, descending=True, stable=True).indices[:top]
        for got, want in ((r.entropy[i], -(lp.exp() * lp).sum()),
                          (r.logprobs[i], torch.stack([lp[k] if k >= 0 else torch.tensor(-math.inf, dtype=torch.float64) for k in t[i]]))):
            far = (got.cpu().double() - want).abs()
            assert ((far <= tol) | (got.cpu().double() == want)).all()
        if top:
            assert torch.equal(r.top_ids[i].cpu().long(), order)
            assert ((r.top_logprobs[i].cpu().double() - lp[order]).abs() <= tol).all()


def test_rotation_of_many_rows_and_heads():
    """Rows past 2^16, and 1024 heads of one row, of sequences that the lengths place anywhere."""
    g = torch.Generator().manual_seed(9)
    for rows, heads, kv, hd in ((70001, 1, 1, 64), (3, 1024, 1024, 64), (2, 3, 1, 256)):
        q, k = (torch.randn(rows, h * hd, generator=g).half() for h in (heads, kv))
        tab = table(rows + 5, 16)
        starts, lens = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([rows + 5], dtype=torch.int32)
        yq, yk = ops.qk_norm_rope(q.cuda(), k.cuda(), hd, tab.cuda(), lens.cuda(), starts.cuda())
        for got, x in ((yq, q), (yk, k)):
            want, tol = rotated(x, None, tab, torch.arange(5, rows + 5), hd, 1e-6)
            tol = tol + HALF[torch.float16] * (want.abs() + tol) + TINY[torch.float16]
            assert ((got.cpu().double().view(want.shape) - want).abs() <= tol).all()
