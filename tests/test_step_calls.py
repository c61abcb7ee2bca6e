"""What the wrappers of the operators around the paged cache hand to the C ABI, on a CPU-only host: a stand-in for the library takes
the calls, and no kernel is there to run."""
from __future__ import annotations

import types

import pytest
import torch

from opentars_amd import ops
from opentars_amd.contract import OUT_BF16, OUT_FP16, OUT_FP32
from test_paged_calls import Far, library, stand_in  # noqa: F401

BIG = 2 ** 32 + 2


class Gpu(Far):
    """A tensor of these sizes that says it is on a GPU."""
    is_cuda, device = True, torch.device("cpu")

    def __init__(self, shape, dtype, ld=None):
        super().__init__(shape, dtype)
        self.ld = ld

    def stride(self, i=None):
        s = (self.shape[1] if self.ld is None else self.ld, 1) if self.dim() == 2 else (1,)
        return s if i is None else s[i]

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()

    def is_contiguous(self):
        return self.ld is None


def weights(n=64, k=512):
    return types.SimpleNamespace(rows=n, cols=k, values=torch.zeros(n, k // 2, dtype=torch.uint8), device=torch.device("cpu"), index=-1,
                                 _ref=None)


def table(positions=10, rot=64):
    return torch.zeros(positions, rot)


@pytest.fixture(autouse=True)
def no_kept_sizes():
    ops._mx4_workspace.cache_clear()
    ops._logprobs_workspace.cache_clear()
    yield
    ops._mx4_workspace.cache_clear()
    ops._logprobs_workspace.cache_clear()


def calls(library):  # noqa: F811
    return [c for c in library.calls if not c[0].endswith("_workspace")]


@pytest.mark.parametrize("out", [2 ** 32, 2 ** 32 + 1, -2 ** 32, 2, -1, 1.5])
def test_products_of_other_outs_are_refused(library, out):  # noqa: F811
    for y in (None, Gpu((2, 64), torch.bfloat16)):
        with pytest.raises(ValueError):
            ops.gemm_mx4(Gpu((2, 512), torch.bfloat16), weights(), out=out, y=y)
    assert not calls(library)


def test_sizes_past_32_bits_are_refused(library):  # noqa: F811
    lens, bf = torch.ones(2, dtype=torch.int32), torch.bfloat16
    for call in (lambda: ops.gemm_mx4(Gpu((BIG, 512), bf), weights(), y=Gpu((BIG, 64), bf)),
                 lambda: ops.token_logprobs(Gpu((2, BIG), bf)),
                 lambda: ops.token_logprobs(Gpu((2, 100), bf), top=2 ** 32 + 5),
                 lambda: ops.token_logprobs(Gpu((2, 100), bf), top=-2 ** 32 + 5),
                 lambda: ops.qk_norm_rope(Far((BIG, 128), bf), Far((BIG, 64), bf), 64, table(), lens, torch.arange(3, dtype=torch.int32),
                                          yq=Far((BIG, 128), bf), yk=Far((BIG, 64), bf)),
                 lambda: ops.qk_norm_rope(torch.zeros(2, 128, dtype=bf), torch.zeros(2, 64, dtype=bf), 64,
                                          Gpu((BIG, 64), torch.float32), lens)):
        with pytest.raises(ValueError):
            call()
    assert not calls(library)


def test_products_hand_on_what_they_are_given(library):  # noqa: F811
    x, w = Gpu((3, 512), torch.bfloat16, 1024), weights()
    ops.gemm_mx4(x, w)
    ops.gemm_mx4(x, w, y=Gpu((3, 64), torch.float32, 80), out=OUT_FP32)
    (a, first), (b, second) = calls(library)
    assert a == b == "tars_quant_gemm_mx4"
    assert first[1:4] == [2048, OUT_BF16, 3] and first[7:9] == [0, OUT_BF16]
    assert second[7:9] == [320, OUT_FP32]
    assert ops.gemm_mx4(Gpu((0, 512), torch.float16), w).shape == (0, 64) and len(calls(library)) == 2
    assert ops.gemm_mx4(Gpu((2, 512), torch.float32), w, out=OUT_FP16).dtype == torch.float16


@pytest.mark.parametrize("kw", [dict(y=Gpu((3, 63), torch.bfloat16)), dict(y=Gpu((3, 64), torch.int8)),
                                dict(y=Gpu((3, 64), torch.bfloat16), out=OUT_FP32), dict(bias=torch.zeros(63)),
                                dict(bias=torch.zeros(64, dtype=torch.float64)), dict(bias=torch.zeros(128)[::2]),
                                dict(y=Gpu((3, 64), torch.bfloat16, 0))])
def test_products_refuse(library, kw):  # noqa: F811
    with pytest.raises(ValueError):
        ops.gemm_mx4(Gpu((3, 512), torch.bfloat16), weights(), **kw)
    for x in (Gpu((3, 480), torch.bfloat16), Gpu((3, 512), torch.int8), Gpu((3, 512), torch.bfloat16, 0), torch.zeros(3, 512)):
        with pytest.raises(ValueError):
            ops.gemm_mx4(x, weights())
    assert not calls(library)


def test_a_matrix_must_hold_whole_blocks():
    for v, s in (((4, 24), (4, 2)), ((4, 16), (4, 2)), ((4, 16), (3, 1)), ((4, 0), (4, 0))):
        with pytest.raises(ValueError):
            ops.Mx4(Gpu(v, torch.uint8), Gpu(s, torch.uint8))
    with pytest.raises(ValueError):
        ops.Mx4(Gpu((4, 16), torch.int8), Gpu((4, 1), torch.uint8))
    with pytest.raises(ValueError):
        ops.Mx4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))   # not on a GPU


def test_rope_hands_on_what_it_is_given(library):  # noqa: F811
    fused = torch.zeros(2, 5 * 64 + 8, dtype=torch.bfloat16)
    lens = torch.ones(2, dtype=torch.int32)
    q, k, v = fused[:, :192], fused[:, 192:256], fused[:, 256:320]
    gamma = torch.ones(64)
    yq, yk = ops.qk_norm_rope(q, k, 64, table(), lens, None, gamma, None, 1e-5, yq=q)
    assert yq is q and yk.shape == k.shape and yk.is_contiguous()
    ops.kv_append_rope(stand_in(), q, k, v, torch.zeros(2, 3, dtype=torch.int32), lens, table(7, 32))
    (a, one), (b, two) = calls(library)
    assert a == "tars_qk_norm_rope" and b == "tars_kv_append_rope"
    assert one[1] == one[3] == 656 and one[4:9] == [0, 3, 1, 64, 2] and one[10] is None and one[13:15] == [10, 64]
    assert one[15] == lens.data_ptr() and one[17:20] == [2, q.data_ptr(), 656] and one[21] == 0
    assert two[2] == two[4] == two[6] == 656 and two[7:10] == [0, 3, 2] and two[14:16] == [7, 32]


@pytest.mark.parametrize("kw", [dict(k=torch.zeros(3, 64, dtype=torch.bfloat16)), dict(k=torch.zeros(2, 64, dtype=torch.float16)),
                                dict(k=torch.zeros(2, 65, dtype=torch.bfloat16)), dict(k=torch.zeros(2, 64)),
                                dict(q=torch.zeros(2, 128, 1, dtype=torch.bfloat16)), dict(hd=0), dict(hd=-64),
                                dict(tab=torch.zeros(10, 64, dtype=torch.float64)), dict(tab=torch.zeros(10, 128)[:, :64]),
                                dict(qgamma=torch.ones(32)), dict(kgamma=torch.ones(64, dtype=torch.bfloat16)),
                                dict(lens=torch.ones(2, dtype=torch.int64)), dict(lens=torch.ones(3, dtype=torch.int32)),
                                dict(starts=torch.zeros(2, dtype=torch.int32)), dict(starts=torch.zeros(3, dtype=torch.int64)),
                                dict(yq=torch.zeros(2, 64, dtype=torch.bfloat16)), dict(yk=torch.zeros(2, 64, dtype=torch.float16)),
                                dict(q=torch.zeros(1, 128, dtype=torch.bfloat16).expand(2, 128))])
def test_rope_refuses(library, kw):  # noqa: F811
    a = dict(q=torch.zeros(2, 128, dtype=torch.bfloat16), k=torch.zeros(2, 64, dtype=torch.bfloat16), hd=64, tab=table(),
             lens=torch.ones(2, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(**a)
    assert not calls(library)


def test_logprobs_hand_on_what_they_are_given(library):  # noqa: F811
    x = Gpu((3, 100), torch.float16, 104)
    r = ops.token_logprobs(x, torch.zeros(3, 5, dtype=torch.int64)[:, 2], top=4)
    assert r.logprobs.shape == (3,) and r.entropy.shape == (3,) and r.top_logprobs.shape == r.top_ids.shape == (3, 4)
    assert r.top_ids.dtype == torch.int32 and r.logprobs.dtype == torch.float32
    assert ops.token_logprobs(x).logprobs is None and ops.token_logprobs(x).top_ids is None
    r = ops.token_logprobs(x, torch.zeros(3, 2, dtype=torch.int32))
    assert r.logprobs.shape == (3, 2)
    first, *_, last = [c[1] for c in calls(library)]
    assert first[1:5] == [208, OUT_FP16, 3, 100] and first[6:9] == [40, 1, 1] and first[11] == 4
    assert last[6:9] == [8, 0, 2] and last[11] == 0
    n = len(calls(library))
    empty = ops.token_logprobs(Gpu((0, 100), torch.float32), torch.zeros(0, dtype=torch.int64), top=2)
    assert empty.logprobs.shape == (0,) and empty.top_ids.shape == (0, 2) and len(calls(library)) == n
    assert ops.token_logprobs(x, torch.zeros(3, 0, dtype=torch.int64)).logprobs.shape == (3, 0)


@pytest.mark.parametrize("kw", [dict(top=65), dict(top=-1), dict(top=101), dict(tokens=torch.zeros(2, dtype=torch.int64)),
                                dict(tokens=torch.zeros(3)), dict(tokens=torch.zeros(3, 1, 1, dtype=torch.int64)),
                                dict(tokens=torch.zeros(1, dtype=torch.int64).expand(3)), dict(tokens=torch.zeros(3, dtype=torch.int16)),
                                dict(tokens=torch.zeros(1, 2, dtype=torch.int64).expand(3, 2))])
def test_logprobs_refuse(library, kw):  # noqa: F811
    a = dict(logits=Gpu((3, 100), torch.bfloat16))
    a.update(kw)
    with pytest.raises(ValueError):
        ops.token_logprobs(**a)
    for logits in (Gpu((3, 100), torch.int8), Gpu((3,), torch.bfloat16), Gpu((3, 100), torch.bfloat16, 0), torch.zeros(3, 100)):
        with pytest.raises(ValueError):
            ops.token_logprobs(logits)
    assert not calls(library)
