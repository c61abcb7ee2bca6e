"""What the paged cache's wrappers hand to the C ABI, on a CPU-only host: a stand-in for the library takes the calls, CPU
tensors stand for the GPU's (both report device -1), and no kernel is there to run."""
from __future__ import annotations

import ctypes
import types

import pytest
import torch

from opentars_amd import _lib, ops
from opentars_amd.contract import OUT_BF16, OUT_FP32


class Library:
    """Takes every call as ctypes would pass it on: integers cut to the declared type's bits."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        types_ = _lib.SIGNATURES[name][1]

        def call(*args):
            assert len(args) == len(types_)
            self.calls.append((name, [t(a).value if t in (ctypes.c_int32, ctypes.c_int64, ctypes.c_float) else a
                                      for t, a in zip(types_, args)]))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    ops._paged_workspace.cache_clear()
    yield lib
    ops._paged_workspace.cache_clear()


def stand_in(**kw):
    return types.SimpleNamespace(**{**dict(index=-1, device=torch.device("cpu"), kv_heads=1, page=16, hd=64, dtype=0, _ref=None), **kw})


def call_args(rows=2):
    return dict(q=torch.zeros(rows, 128, dtype=torch.bfloat16), table=torch.zeros(rows, 3, dtype=torch.int32),
                lens=torch.ones(rows, dtype=torch.int32))


@pytest.mark.parametrize("kw", [dict(out=2 ** 32), dict(out=2 ** 32, y=torch.zeros(2, 128, dtype=torch.bfloat16)),
                                dict(out=2 ** 32 + 1), dict(out=-2 ** 32), dict(window=2 ** 32 + 5), dict(window=2 ** 31),
                                dict(window=5 - 2 ** 32), dict(sinks=2 ** 32), dict(sinks=2 ** 40 + 3), dict(sinks=-2 ** 33)])
def test_integers_past_32_bits_are_refused(library, kw):
    """ctypes would cut them: out = 2^32 to FP32 (0), four bytes for each two of y's; a window of 2^32 + 5 to one of 5."""
    a = call_args()
    with pytest.raises(ValueError):
        ops.paged_decode(stand_in(), **a, **kw)
    with pytest.raises(ValueError):
        ops.paged_attention(stand_in(), **a, starts=torch.arange(3, dtype=torch.int32), **kw)
    assert not [n for n, _ in library.calls if n != "tars_paged_workspace"]


class Far:
    """A tensor of these sizes, for shapes that no test can allocate."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype = shape, dtype

    def get_device(self):
        return -1

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape[0] * (self.shape[1] if self.dim() > 1 else 1)

    def stride(self, i=None):
        s = (self.shape[1], 1) if self.dim() == 2 else (1,)
        return s if i is None else s[i]

    def data_ptr(self):
        return 1 << 40


def test_sizes_past_32_bits_are_refused(library):
    """2^32 + 4 pages of a table row would be four, 2^32 + 2 sequences two."""
    q = torch.zeros(2, 128, dtype=torch.bfloat16)
    wide, lens = Far((2, 2 ** 32 + 4), torch.int32), torch.ones(2, dtype=torch.int32)
    n = 2 ** 32 + 2
    many = dict(table=Far((n, 1), torch.int32), lens=Far((n,), torch.int32))
    for call in (lambda: ops.paged_decode(stand_in(), q, wide, lens), lambda: ops.kv_append(stand_in(), q[:, :64], q[:, :64], wide, lens),
                 lambda: ops.paged_attention(stand_in(), q, **many, starts=Far((n + 1,), torch.int32)),
                 lambda: ops.kv_append(stand_in(), q[:, :64], q[:, :64], **many, starts=Far((n + 1,), torch.int32)),
                 lambda: ops.kv_append(stand_in(), Far((n, 64), torch.bfloat16), Far((n, 64), torch.bfloat16), call_args()["table"],
                                       lens, torch.arange(3, dtype=torch.int32)),
                 lambda: ops.paged_attention(stand_in(), Far((n, 128), torch.bfloat16), call_args()["table"], lens,
                                             torch.arange(3, dtype=torch.int32), y=Far((n, 128), torch.bfloat16))):
        with pytest.raises(ValueError):
            call()
    assert not library.calls


def test_a_pool_of_sizes_past_32_bits_is_refused(library):
    """2^32 + 1 pages that are one and the same would be a pool of one page."""
    page = types.SimpleNamespace(is_cuda=True, device=torch.device("cpu"), dtype=torch.bfloat16, shape=(2 ** 32 + 1, 1, 16, 64),
                                 dim=lambda: 4, numel=lambda: 2 ** 42, stride=lambda i=None: (0, 1024, 64, 1) if i is None else 1,
                                 get_device=lambda: -1, element_size=lambda: 2, data_ptr=lambda: 1 << 40)
    with pytest.raises(ValueError):
        ops.PagedCache(page, page)


def test_what_fits_is_passed_on(library):
    a = call_args()
    y = ops.paged_decode(stand_in(), **a, window=2 ** 31 - 1, sinks=2 ** 31 - 1, out=OUT_FP32)
    ops.paged_attention(stand_in(), **a, starts=torch.arange(3, dtype=torch.int32), window=7, sinks=4)
    ops.kv_append(stand_in(), a["q"][:, :64], a["q"][:, 64:], a["table"], a["lens"])
    decode, prompt, store = [c for c in library.calls if c[0] != "tars_paged_workspace"]
    assert y.dtype == torch.float32
    assert decode[0] == "tars_paged_decode" and decode[1][8] == OUT_FP32 and decode[1][10:12] == [2 ** 31 - 1] * 2
    assert prompt[0] == "tars_paged_attention" and prompt[1][8] == OUT_BF16 and prompt[1][10:12] == [7, 4]
    assert store[0] == "tars_kv_append" and store[1][6] == 2 and store[1][2] == 256


@pytest.mark.parametrize("decode", [0, 1])
def test_no_workspace_for_sizes_that_the_calls_refuse(decode):
    size = _lib.lib().tars_paged_workspace
    good = dict(heads=8, kv=2, hd=128, rows=3, seqs=3, width=4096, page=16)
    assert size(*good.values(), decode) > 0
    for bad in (dict(hd=32), dict(hd=96), dict(hd=512), dict(hd=1), dict(page=3), dict(page=1), dict(page=8), dict(page=48),
                dict(page=-16), dict(kv=3), dict(kv=0), dict(heads=1026), dict(rows=0), dict(rows=2 ** 22 + 1), dict(seqs=65536),
                dict(width=2 ** 27), dict(width=0), dict(heads=1024, rows=2 ** 19), dict(heads=1024, seqs=4097)):
        assert size(*{**good, **bad}.values(), decode) == 0, bad
