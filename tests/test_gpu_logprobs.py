"""Log probabilities, entropy and top alternatives on the GPU (ops.token_logprobs) against their definition in 64 bits. Needs a
gfx950 GPU."""
from __future__ import annotations

import math

import pytest
import torch

from opentars_amd import _lib, ops
from step_data import logprobs

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def close(got, want, size, n):
    """fp32 steps: the differences to the maximum and their exponentials (8, of a size of up to `size`), the sum's n terms in
    lanes (2 sqrt(n), on average), the logarithm."""
    got, want = torch.as_tensor(got, dtype=torch.float64), torch.as_tensor(want, dtype=torch.float64)
    tol = (16 + 2 * math.sqrt(n)) * 2.0 ** -24 + 8 * 2.0 ** -24 * size
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert (same | ((got - want).abs() <= tol)).all(), (got, want, tol)


def check(x, tokens, top, xg=None, wide=torch.int64):
    t = None if tokens is None else torch.tensor(tokens, dtype=wide)
    r = ops.token_logprobs(x.cuda() if xg is None else xg, None if t is None else t.cuda(), top=top)
    for i in range(x.shape[0]):
        mine = [] if t is None else t.reshape(x.shape[0], -1)[i].tolist()
        given, h, tv, ti = logprobs(x[i], mine, top)
        ok = x[i][torch.isfinite(x[i])].double()
        size = float(ok.max() - ok.min()) if ok.numel() else 0.0
        if t is not None:
            close(r.logprobs.cpu().view(x.shape[0], -1)[i], given, size, x.shape[1])
        close(r.entropy[i].cpu(), h, 20.0, x.shape[1])
        if top:
            assert r.top_ids[i].tolist() == ti
            close(r.top_logprobs[i].cpu(), tv, size, x.shape[1])
    return r


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 64, 64), (5, 1000, 20), (2, 4099, 64), (1, 33333, 5),
                                            (4, 16384, 1), (70, 515, 3), (3, 2048, 0)])
def test_random_rows(t, rows, vocab, top):
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(TYPES[t])
    tokens = torch.randint(0, vocab, (rows, 3), generator=g).tolist()
    check(x, tokens, top)


@pytest.mark.parametrize("rows", [1, 3, 300])
def test_many_rows_and_parts_of_rows_give_the_same(rows):
    """A row's answer in a call of its own, split over workgroups, and among others."""
    g = torch.Generator().manual_seed(rows)
    x = (4 * torch.randn(rows, 50001, generator=g)).to(torch.bfloat16).cuda()
    t = torch.randint(0, 50001, (rows,), generator=g).cuda()
    all_ = ops.token_logprobs(x, t, top=10)
    for i in {0, rows // 2, rows - 1}:
        one = ops.token_logprobs(x[i:i + 1], t[i:i + 1], top=10)
        assert torch.equal(one.top_ids[0], all_.top_ids[i])
        close(one.top_logprobs[0].cpu(), all_.top_logprobs[i].cpu(), 40.0, 50001)
        close(one.logprobs.cpu(), all_.logprobs[i:i + 1].cpu(), 40.0, 50001)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("lead", [0, 1, 3, 5, 8])
def test_rows_at_any_element(t, lead):
    """Views whose rows start and end inside a 16-byte piece; what lies around them is NaN."""
    g = torch.Generator().manual_seed(lead)
    for vocab in (1, 2, 9, 31, 1024, 5003):
        wide = torch.full((4, vocab + 19), math.nan, dtype=TYPES[t])
        wide[:, lead:lead + vocab] = (2 * torch.randn(4, vocab, generator=g)).to(TYPES[t])
        w = wide.cuda()
        check(wide[:, lead:lead + vocab], [[0, vocab - 1]] * 4, min(vocab, 7), xg=w[:, lead:lead + vocab])


@pytest.mark.parametrize("top", [1, 3, 64])
def test_equal_logits_come_by_their_places(top):
    x = torch.zeros(1, 3000)
    assert check(x, [[0, 2999]], top).top_ids[0].tolist() == list(range(top))
    x[0, 5::7] = 1.0
    check(x, None, top)
    x[0] = -math.inf
    check(x, [[3, 4]], top)                                            # nothing can come
    x[0, 100] = -5.0
    check(x, [[3, 100]], top)
    x[0, 2000:2002] = torch.tensor([-0.0, 0.0])                       # equal
    check(x, None, top)
    x = torch.randint(0, 3, (3, 40000)).float()
    check(x, [[1], [2], [3]], top)


@pytest.mark.parametrize("up", [True, False])
def test_rows_in_order(up):
    """Every logit passes the list's last one, or none after the first."""
    x = torch.arange(20000, dtype=torch.float32)[None] * 1e-3
    x = x if up else x.flip(1).contiguous()
    check(x, [[0, 19999]], 64)


def test_masks_of_the_types_lowest_value():
    g = torch.Generator().manual_seed(2)
    for t in TYPES.values():
        x = torch.randn(2, 5000, generator=g).to(t)
        x[0, torch.rand(5000, generator=g) < 0.9] = torch.finfo(t).min
        x[1] = torch.finfo(t).min
        r = ops.token_logprobs(x.cuda(), torch.tensor([3, 4]).cuda(), top=5)
        assert torch.isfinite(r.entropy).all()
        assert abs(float(r.entropy[1]) - math.log(5000)) < 1e-5 and r.top_ids[1].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("where", [0, 77, 9999])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nan_and_infinity_make_the_row_nan(where, bad):
    g = torch.Generator().manual_seed(where)
    x = torch.randn(3, 10000, generator=g)
    x[1, where] = bad
    r = ops.token_logprobs(x.cuda(), torch.tensor([[5, -1]] * 3).cuda(), top=4)
    assert torch.isnan(r.logprobs[1, 0]) and r.logprobs[1, 1] == -math.inf and torch.isnan(r.entropy[1])
    assert torch.isnan(r.top_logprobs[1]).all() and r.top_ids[1, 0] == where
    for i in (0, 2):
        given, h, tv, ti = logprobs(x[i], [5, -1], 4)
        close(r.logprobs[i].cpu(), given, 10.0, 10000)
        assert r.top_ids[i].tolist() == ti
    x[1] = math.nan
    assert ops.token_logprobs(x.cuda(), top=64).top_ids[1].tolist() == list(range(64))


def test_tokens_of_both_types_shapes_and_outside():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 300, generator=g)
    for wide in (torch.int32, torch.int64):
        check(x, [0, 299, 300, -1], 0, wide=wide)
        check(x, [[0, 299, 300, -1, 7]] * 4, 2, wide=wide)
    wide = torch.tensor([[1, 2, 3, 4], [5, 6, 7, 8], [9, 10, 11, 12], [13, 14, 15, 16]])
    a = ops.token_logprobs(x.cuda(), wide.cuda()[:, 1])
    b = ops.token_logprobs(x.cuda(), wide.cuda()[:, 1:3])
    assert torch.equal(a.logprobs, b.logprobs[:, 0]) and torch.equal(a.logprobs, ops.token_logprobs(x.cuda(), wide[:, 1].cuda()).logprobs)
    big = torch.tensor([2 ** 32, 2 ** 40 + 3, -2 ** 40, 2 ** 63 - 1])
    assert (ops.token_logprobs(x.cuda(), big.cuda()).logprobs == -math.inf).all()
    assert ops.token_logprobs(x.cuda(), torch.zeros(4, 0, dtype=torch.int64).cuda()).logprobs.shape == (4, 0)
    assert ops.token_logprobs(x[:0].cuda(), top=3).top_ids.shape == (0, 3)


def test_far_logits():
    """Logits far from zero and from each other: differences, not exponentials, are what is kept."""
    x = torch.tensor([[3e38, 2.9e38, -3e38, 0.0], [-3.4e38, -3.4e38, -3.4e38, -3.4e38], [1e30, 1e30, 0, 0], [5e4, 5e4 - 1, 5e4 - 2, -6e4]])
    r = ops.token_logprobs(x.cuda(), torch.zeros(4, dtype=torch.int64).cuda(), top=4)
    want = torch.tensor([0.0, -math.log(4), -math.log(2), -math.log(1 + math.exp(-1) + math.exp(-2))])
    assert ((r.logprobs.cpu() - want).abs() < 1e-6).all() and torch.isfinite(r.entropy).all()


def test_rows_past_4_gib():
    x = torch.zeros(17, 1 << 26, dtype=torch.float32, device="cuda")[:, :1 << 24]          # rows 256 MiB apart
    x[16, (1 << 24) - 1] = 30.0
    r = ops.token_logprobs(x, torch.full((17,), (1 << 24) - 1, device="cuda"), top=1)
    want = 30 - math.log(math.exp(30) + (1 << 24) - 1)
    assert abs(float(r.logprobs[16]) - want) < 1e-5 and int(r.top_ids[16, 0]) == (1 << 24) - 1 and int(r.top_ids[15, 0]) == 0


@pytest.mark.parametrize("rows", [1, 40])
def test_streams_and_graphs(rows):
    g = torch.Generator().manual_seed(rows)
    xs = [torch.randn(rows, 30011, generator=g).cuda() for _ in range(3)]
    t = torch.randint(0, 30011, (rows,), generator=g).cuda()
    eager = [ops.token_logprobs(x, t, top=6) for x in xs]
    buf = xs[0].clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.token_logprobs(buf, t, top=6)
    for i in (1, 0, 2, 1):
        buf.copy_(xs[i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = ops.token_logprobs(xs[(i + 1) % 3], t, top=6)
        torch.cuda.synchronize()
        for got, want in ((r, eager[i]), (other, eager[(i + 1) % 3])):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x = torch.zeros(2, 50, device="cuda")
    for call in (lambda: ops.token_logprobs(x, top=51), lambda: ops.token_logprobs(x, top=-1), lambda: ops.token_logprobs(x.int()),
                 lambda: ops.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda")), lambda: ops.token_logprobs(x.T),
                 lambda: ops.token_logprobs(x, torch.zeros(2, device="cuda")), lambda: ops.token_logprobs(x.cpu()),
                 lambda: ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64)), lambda: ops.token_logprobs(x[0]),
                 lambda: ops.token_logprobs(x[:1].expand(2, 50))):
        with pytest.raises((ValueError, ops.TarsError)):
            call()


def test_the_workspace_ends_where_it_says():
    lib = _lib.lib()
    for rows, vocab, top in ((1, 151936, 5), (7, 60001, 64), (300, 9000, 0)):
        x = torch.randn(rows, vocab, device="cuda")
        need = lib.tars_logprobs_workspace(rows, vocab, 0, top)
        room = torch.full((need + 512,), 0x5A, dtype=torch.uint8, device="cuda")
        h = torch.empty(rows, device="cuda")
        tv, ti = torch.empty(rows, max(top, 1), device="cuda"), torch.empty(rows, max(top, 1), dtype=torch.int32, device="cuda")
        rc = lib.tars_token_logprobs(x.data_ptr(), 0, 0, rows, vocab, None, 0, 0, 0, None, h.data_ptr(), top, tv.data_ptr(), ti.data_ptr(),
                                     room.data_ptr() + 256, need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.last_error()
        want = ops.token_logprobs(x, top=top)
        assert torch.equal(h, want.entropy) and (not top or torch.equal(ti, want.top_ids))
        assert (room[:256] == 0x5A).all() and (room[256 + need:] == 0x5A).all()
