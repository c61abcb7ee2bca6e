"""Microscaled 4-bit floating point on the GPU (ops.Mx4, quant_mx4, gemm_mx4) against its definition in 64 bits. Needs a
gfx950 GPU."""
from __future__ import annotations

import math

import pytest
import torch

from opentars_amd import _lib, ops
from opentars_amd.contract import OUT_BF16, OUT_FP16, OUT_FP32
from step_data import HALF, TINY, packed, quantised, random_codes, values_of

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
OUT = {"bf16": OUT_BF16, "fp16": OUT_FP16, "fp32": OUT_FP32}


def bits(t):
    return t.view(torch.int32 if t.element_size() == 4 else torch.int16)


def check_codes(m, x):
    code, byte = quantised(x)
    code = torch.where(byte.repeat_interleave(32, 1) == 255, 0, code)
    assert torch.equal(m.scales.cpu().int(), byte.int())
    assert torch.equal(m.values.cpu(), packed(code))


# ------------------------------------------------------------------------------------------------ quant_mx4
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (5, 2080), (70, 512), (2, 16384)])
def test_quant_of_random_rows(t, rows, cols):
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-9, 9, (rows, cols), generator=g).float())
    x = x.to(TYPES[t])
    m = ops.quant_mx4(x.cuda())
    check_codes(m, x)
    pieces = m.scales.as_strided((rows, -(-cols // 512) * 16), m.scales.stride()).cpu()
    assert not pieces[:, cols // 32:].any()                       # the padded row's end


@pytest.mark.parametrize("t", TYPES)
def test_quant_of_every_kind_of_block(t):
    """Ties, zeros of both signs, subnormals, the type's ends, and infinities or NaN in one block beside others."""
    dt = TYPES[t]
    info = torch.finfo(dt)
    x = torch.zeros(12, 96, dtype=torch.float64)
    ticks = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, .125, .24, .26, .74, .76, 1.24, 1.26, 2.4,
                          2.6, 3.4, 3.6, 4.9, 5.1, 6.9, 7.5, 4.5])
    x[0, :32], x[0, 32:64] = ticks, -ticks
    x[1, :32], x[1, 64:] = ticks * 2 ** -10, -ticks * 2 ** 10
    x[2, 5], x[2, 40], x[2, 70] = info.max, -info.max, info.tiny
    x[3, 1] = info.smallest_normal / 8                             # subnormal
    x[4, :32] = ticks * info.smallest_normal
    x[5, 3], x[5, 70] = math.inf, 1.0
    x[6, 33], x[6, 64] = math.nan, -2.5
    x[7, 0], x[7, 31], x[7, 32] = -math.inf, math.nan, 3.0
    x[8] = -0.0
    x[9, 0], x[9, 1] = 1.0, -2.0 ** -14                             # rounds to -0
    x[10, ::3] = -info.smallest_normal
    x[11] = 1 / 3
    x = x.to(dt)
    check_codes(ops.quant_mx4(x.cuda()), x)


def test_quant_of_strided_rows_and_none():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(9, 640, generator=g).half()
    w = wide.cuda()
    check_codes(ops.quant_mx4(w[:, 64:384]), wide[:, 64:384])
    check_codes(ops.quant_mx4(w[::2, :96]), wide[::2, :96])
    check_codes(ops.quant_mx4(w[3:4, 8:40]), wide[3:4, 8:40])
    m = ops.quant_mx4(w[:0])
    assert m.rows == 0 and m.cols == 640


# ------------------------------------------------------------------------------------------------ gemm_mx4
def exact_case(seed, M, N, K):
    """Codes whose products are whole quarters and whose sums stay below 2^24 of them: fp32 holds every sum exactly."""
    g = torch.Generator().manual_seed(seed)
    x, w = random_codes(g, M, K), random_codes(g, N, K)
    return x, w, values_of(*x) @ values_of(*w).T


def dev(code, byte):
    return ops.Mx4(packed(code).cuda(), byte.to(torch.uint8).cuda())


SHAPES = [(1, 1, 32), (1, 16, 128), (1, 2048, 1024), (2, 5, 96), (1, 257, 4096), (3, 33, 160), (16, 64, 256), (17, 48, 512), (33, 70, 1056),
          (64, 129, 544), (65, 16, 64), (100, 1, 32), (128, 128, 256), (129, 257, 288), (200, 333, 1024), (256, 256, 2048),
          (300, 1030, 736), (1, 5000, 64), (37, 1536, 1536), (515, 100, 96), (1000, 31, 320), (257, 4097, 32)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_sums_that_fp32_holds_are_exact(M, N, K):
    x, w, want = exact_case(M * 7 + N + K, M, N, K)
    got = ops.gemm_mx4(dev(*x), dev(*w), out=OUT_FP32)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("M,N,K", [(1, 40, 256), (9, 130, 96), (40, 64, 512), (70, 515, 288), (260, 300, 256)])
@pytest.mark.parametrize("out", OUT)
def test_outputs_bias_and_strides(M, N, K, out):
    x, w, want = exact_case(M + N, M, N, K)
    g = torch.Generator().manual_seed(5)
    bias = torch.randn(N, generator=g)
    dt = TYPES[out]
    want = (want + bias.double())
    for lead, gap in ((0, 0), (4, 8), (1, 2), (0, 3)):                # aligned rows and others, the gaps left as they were
        room = torch.full((M, lead + N + gap), 7.0, dtype=dt, device="cuda")
        y = room[:, lead:lead + N]
        assert ops.gemm_mx4(dev(*x), dev(*w), bias=bias.cuda(), y=y) is y
        # the sum is exact, the bias one fp32 step, the output another
        tol = 2 ** -24 * want.abs() + HALF[dt] * (1 + 2 ** -23) * want.abs() + TINY[dt]
        if dt == torch.float16:
            assert want.abs().max() < 65000
        assert ((y.cpu().double() - want).abs() <= tol).all()
        rest = room.clone()
        rest[:, lead:lead + N] = 7.0
        assert (rest == 7.0).all()


@pytest.mark.parametrize("M,N,K", [(112, 11, 4352), (100, 1024, 8192), (97, 200, 10272), (842, 194, 4128), (130, 64, 16384)])
def test_few_tiles_with_k_in_parts(M, N, K):
    """A long K for few tiles is summed in parts: their sums in fp32 are whole quarters too, whichever part holds a k."""
    x, w, want = exact_case(M + N + K, M, N, K)
    a, b = dev(*x), dev(*w)
    bias = (torch.arange(N) % 16 - 8).float()
    assert _lib.lib().tars_mx4_workspace(M, N, K, 0) > 0
    assert torch.equal(ops.gemm_mx4(a, b, out=OUT_FP32).cpu().double(), want)
    for out, lead in ((OUT_FP32, 1), (OUT_BF16, 0), (OUT_FP16, 3)):
        dt = TYPES["bf16" if out == OUT_BF16 else "fp16" if out == OUT_FP16 else "fp32"]
        room = torch.full((M, lead + N + 5), 7.0, dtype=dt, device="cuda")
        ops.gemm_mx4(a, b, bias=bias.cuda(), y=room[:, lead:lead + N])
        assert torch.equal(room[:, lead:lead + N].cpu(), (want + bias.double()).to(dt))
        room[:, lead:lead + N] = 7.0
        assert (room == 7.0).all()
    x[1][5, K // 32 - 1] = 255                                        # NaN in the last part alone
    y = ops.gemm_mx4(dev(*x), b, out=OUT_FP32).cpu()
    assert torch.isnan(y[5]).all() and torch.equal(y[:5].double(), want[:5]) and torch.equal(y[6:].double(), want[6:])


@pytest.mark.parametrize("M,N,K,lead", [(2011, 12288, 4096, 0), (2011, 12301, 4096, 3), (1200, 20000, 2048, 0)])
def test_more_tiles_than_a_round(M, N, K, lead):
    """Every 64th column, those around tiles' ends, the last."""
    x, w = (random_codes(torch.Generator().manual_seed(M + n), n, K) for n in (M, N))
    bias = (torch.arange(N) % 16 - 8).float()
    room = torch.full((M, lead + N + 5), 7.0, dtype=torch.float32, device="cuda")
    ops.gemm_mx4(dev(*x), dev(*w), bias=bias.cuda(), y=room[:, lead:lead + N])
    at = torch.tensor([n for n in range(N) if n % 64 == 5 or n % 128 in (0, 127) or n > N - 20])
    want = values_of(*x).float() @ values_of(w[0][at], w[1][at]).float().T + bias[at]     # exact: whole quarters below 2^24 of them
    assert torch.equal(room[:, lead:lead + N].cpu()[:, at], want)
    room[:, lead:lead + N] = 7.0
    assert (room == 7.0).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 64, 1024), (5, 33, 96), (16, 100, 4096), (17, 40, 288), (64, 64, 64), (90, 200, 512), (1, 3000, 512)])
def test_a_tensor_is_quantised_in_the_call(t, M, N, K):
    g = torch.Generator().manual_seed(M * N + K)
    x = torch.randn(M, K + 16, generator=g) * torch.where(torch.rand(K + 16, generator=g) < 0.05, 20.0, 1.0)
    x = x.to(TYPES[t])
    w = random_codes(g, N, K, low=118, spread=4)
    xg = x.cuda()[:, 16:] if t != "fp32" else x.cuda()[:, 4:K + 4]
    xc = xg.cpu()
    q = ops.quant_mx4(xg)
    check_codes(q, xc)
    a, b = values_of(*quantised(xc)), values_of(*w)
    want, size = a @ b.T, a.abs() @ b.abs().T
    got = ops.gemm_mx4(xg, dev(*w))
    assert got.dtype == x.dtype
    tol = (8 + 2 * math.sqrt(K)) * 2.0 ** -24 * size
    tol += HALF[x.dtype] * (want.abs() + tol) + TINY[x.dtype]
    assert ((got.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(bits(got), bits(ops.gemm_mx4(q, dev(*w), out=OUT[t])))  # the same in two calls


def test_scales_over_the_whole_range():
    """Exponents at either end, products within fp32: the instruction's sums of exponents, not the scales as numbers."""
    g = torch.Generator().manual_seed(3)
    for lo_x, lo_w in ((0, 200), (250, 4), (1, 130), (127, 127), (254, 0)):
        x, w = random_codes(g, 20, 256, low=lo_x, spread=1), random_codes(g, 30, 256, low=lo_w, spread=1)
        want = values_of(*x) @ values_of(*w).T
        assert torch.equal(ops.gemm_mx4(dev(*x), dev(*w), out=OUT_FP32).cpu().double(), want)


@pytest.mark.parametrize("M", [1, 20, 80, 300])
def test_nan_blocks_reach_their_rows_and_columns_alone(M):
    K, N = 544, 70
    x, w, want = exact_case(M, M, N, K)
    x[1][M // 2, 16] = 255
    w[1][33, 0] = 255
    y = ops.gemm_mx4(dev(*x), dev(*w), out=OUT_FP32).cpu().double()
    want[M // 2] = math.nan
    want[:, 33] = math.nan
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(y, nan=0), torch.nan_to_num(want, nan=0))


@pytest.mark.parametrize("M", [1, 40, 200])
def test_what_lies_behind_k_is_not_read_into_a_sum(M):
    """Rows of a wider matrix whose neighbours are NaN blocks: k ends inside a piece of 128, of 512 and of a scales' 16 bytes."""
    g = torch.Generator().manual_seed(M)
    for K in (32, 96, 160, 480, 800):
        wide = 1536
        x, w = random_codes(g, M, wide), random_codes(g, 50, wide)
        x[1][:, K // 32:], w[1][:, K // 32:] = 255, 255
        vx, vw = packed(x[0]).cuda(), packed(w[0]).cuda()
        sx, sw = x[1].to(torch.uint8).cuda(), w[1].to(torch.uint8).cuda()
        mx, mw = (ops.Mx4(v[:, :K // 2], s[:, :K // 32]) for v, s in ((vx, sx), (vw, sw)))
        assert mx.values.data_ptr() == vx.data_ptr() and mw.scales.data_ptr() == sw.data_ptr()    # the views themselves
        want = values_of(x[0][:, :K], x[1][:, :K // 32]) @ values_of(w[0][:, :K], w[1][:, :K // 32]).T
        assert torch.equal(ops.gemm_mx4(mx, mw, out=OUT_FP32).cpu().double(), want)


def test_matrices_that_do_not_lie_right_are_laid_out():
    g = torch.Generator().manual_seed(8)
    x, w = random_codes(g, 3, 96), random_codes(g, 40, 96)
    want = values_of(*x) @ values_of(*w).T
    v = torch.zeros(40, 49, dtype=torch.uint8)
    v[:, 1:] = packed(w[0])
    s = torch.zeros(3, 40, dtype=torch.uint8)
    s[:] = w[1].T
    m = ops.Mx4(v.cuda()[:, 1:], s.cuda().T)
    for a in (dev(*x), ops.Mx4(packed(x[0]).cuda().T.contiguous().T, x[1].to(torch.uint8).cuda())):
        assert torch.equal(ops.gemm_mx4(a, m, out=OUT_FP32).cpu().double(), want)


def test_an_all_nan_row_and_zero_rows_of_a_batch():
    g = torch.Generator().manual_seed(9)
    w = random_codes(g, 64, 128)
    x = torch.randn(6, 128, generator=g).bfloat16()
    x[2], x[4], x[5, 7] = 0, math.nan, math.inf
    y = ops.gemm_mx4(x.cuda(), dev(*w), out=OUT_FP32).cpu()
    assert (y[2] == 0).all() and torch.isnan(y[4]).all() and torch.isnan(y[5]).all() and torch.isfinite(y[[0, 1, 3]]).all()
    assert ops.gemm_mx4(x[:0].cuda(), dev(*w)).shape == (0, 64)


def test_past_binary16_is_infinity():
    x = (torch.full((1, 32), 7), torch.full((1, 1), 135))              # 6 * 2^8
    w = (torch.full((2, 32), 7), torch.tensor([[135], [120]]))
    y = ops.gemm_mx4(dev(*x), dev(*w), out=OUT_FP16).cpu()
    assert y[0, 0] == math.inf and y[0, 1] == 32 * 36 * 2.0


@pytest.mark.parametrize("M", [1, 30, 150])
def test_streams_and_graphs(M):
    """A captured product replayed with other rows, between eager calls of the same sizes on another stream."""
    g = torch.Generator().manual_seed(M)
    w = dev(*random_codes(g, 300, 512))
    xs = [torch.randn(M, 512, generator=g).bfloat16().cuda() for _ in range(3)]
    eager = [ops.gemm_mx4(x, w) for x in xs]
    buf, y = xs[0].clone(), torch.empty(M, 300, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.gemm_mx4(buf, w, y=y)
    for i in (1, 2, 0, 1):
        buf.copy_(xs[i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = ops.gemm_mx4(xs[(i + 1) % 3], w)
        torch.cuda.synchronize()
        assert torch.equal(bits(y), bits(eager[i])) and torch.equal(bits(other), bits(eager[(i + 1) % 3]))


@pytest.mark.parametrize("bad", ["dtype", "k", "cols", "bias", "y", "out", "cpu", "place"])
def test_refusals(bad):
    g = torch.Generator().manual_seed(1)
    w, x = dev(*random_codes(g, 64, 128)), torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    kw = {}
    if bad == "dtype":
        x = x.int()
    elif bad == "k":
        x = x[:, :96]
    elif bad == "cols":
        with pytest.raises(ValueError):
            ops.quant_mx4(x[:, :40])
        return
    elif bad == "bias":
        kw["bias"] = torch.zeros(65, device="cuda")
    elif bad == "y":
        kw["y"] = torch.zeros(2, 63, dtype=torch.bfloat16, device="cuda")
    elif bad == "out":
        kw["out"] = 2
    elif bad == "cpu":
        x = x.cpu()
    else:
        kw["y"] = x.view(torch.bfloat16)[:, :64]
    with pytest.raises((ValueError, ops.TarsError)):
        ops.gemm_mx4(x, w, **kw)


def test_the_workspace_ends_where_it_says():
    lib = _lib.lib()
    g = torch.Generator().manual_seed(2)
    for M, N, K in ((40, 64, 288), (200, 300, 4096), (70, 33, 8192), (300, 130, 96)):
        code, byte = random_codes(g, N, K)
        w, x = dev(code, byte), torch.randn(M, K, generator=g).bfloat16().cuda()
        need = lib.tars_mx4_workspace(M, N, K, 1)
        room = torch.full((need + 512,), 0x5A, dtype=torch.uint8, device="cuda")
        y = torch.empty(M, N, dtype=torch.bfloat16, device="cuda")
        rc = lib.tars_quant_gemm_mx4(x.data_ptr(), 0, OUT_BF16, M, w._ref, None, y.data_ptr(), 0, OUT_BF16, room.data_ptr() + 256, need,
                                     torch.cuda.current_stream().cuda_stream)
        assert rc == 0, _lib.last_error()
        assert torch.equal(bits(y), bits(ops.gemm_mx4(x, w)))
        assert (room[:256] == 0x5A).all() and (room[256 + need:] == 0x5A).all()


@pytest.mark.parametrize("M,N,K", [(16, 600, 5120), (37, 515, 1536), (64, 256, 4096), (100, 1024, 8192), (300, 300, 1056)])
def test_a_rows_bits_are_its_own(M, N, K):
    """At the same sizes a row's result has the same bits wherever it is and whatever the other rows are. The scales are far enough
    apart (2^30) that fp32 rounds the sums."""
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, K, generator=g).bfloat16()
    codes = random_codes(g, N, K, low=100, spread=30)
    w = dev(*codes)
    y = ops.gemm_mx4(x.cuda(), w, out=OUT_FP32).cpu()
    exact = values_of(*quantised(x)) @ values_of(*codes).T
    assert (y.double() != exact).double().mean() > 0.5
    order = torch.randperm(M, generator=g)
    assert torch.equal(bits(ops.gemm_mx4(x[order].cuda(), w, out=OUT_FP32).cpu()), bits(y[order]))
    other = torch.randn(M, K, generator=g).bfloat16()
    other[M // 3] = x[M // 3]
    assert torch.equal(bits(ops.gemm_mx4(other.cuda(), w, out=OUT_FP32).cpu()[M // 3]), bits(y[M // 3]))


# ------------------------------------------------------------------------------------------------ few rows, the ways through w
# Several loads of a wave's share of K to a tile of w, K ending inside the last one; waves without a share; a workgroup's second
# tiles, with and without waves that share one; one, two and three groups of 16 rows.
FEW = [(1, 80, 5120), (1, 64, 10336), (3, 6001, 5120), (16, 6000, 2560), (16, 9728, 2560), (16, 12288, 4096), (5, 2100, 5152), (17, 5120, 2560),
       (24, 1000, 3616), (20, 70000, 1056), (2, 66000, 544), (33, 70000, 288), (37, 12288, 1536), (48, 300, 1568), (48, 200, 2560)]


def few_case(M, N, K):
    """Codes of sums that are whole quarters below 2^24 of them, in fp32 too; NaN in the last block of a row of each."""
    g = torch.Generator().manual_seed(M + N + K)
    x, w = random_codes(g, M, K), random_codes(g, N, K)
    a, b = values_of(*x).float(), values_of(*w).float()
    want = a @ b.T
    w[1][N // 2, -1] = 255
    want[:, N // 2] = math.nan
    return x, w, a, want


@pytest.mark.parametrize("M,N,K", FEW)
def test_few_rows_of_a_long_k_and_of_many_columns(M, N, K):
    x, w, _, want = few_case(M, N, K)
    wd = dev(*w)
    bias = (torch.arange(N) % 16 - 8).float()
    got = ops.gemm_mx4(dev(*x), wd, bias=bias.cuda(), out=OUT_FP32).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want + bias, nan=1e9))
    x[1][M // 2, -1] = 255
    want[M // 2] = math.nan
    got = ops.gemm_mx4(dev(*x), wd, out=OUT_FP32).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 80, 5120), (16, 9728, 2560), (16, 1000, 5120), (17, 5120, 2560), (37, 12288, 1536), (48, 200, 2560)])
def test_few_rows_quantised_by_the_product_itself(t, M, N, K):
    """Values of four bits come back as themselves: a block whose largest is 3 or less has a smaller scale and the same values."""
    _, w, a, want = few_case(M, N, K)
    assert _lib.lib().tars_mx4_workspace(M, N, K, 1) == 0             # no launch before it
    x = a.to(TYPES[t])
    assert torch.equal(x.float(), a)
    got = ops.gemm_mx4(x.cuda(), dev(*w), out=OUT_FP32).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))
