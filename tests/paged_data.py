"""A paged key / value cache for tests: pools whose unused slots hold NaN, tables whose unused entries name no page, and
the attention's definition in 64 bits with the error that its roundings allow."""
from __future__ import annotations

import math

import torch

QT = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
E4M3 = torch.float8_e4m3fn


def empty_pool(pages, kv, page, hd, dtype, layout="hnd"):
    """K and V pools [pages, kv, page, hd] full of NaN: heads outside slots ("hnd"), slots outside heads ("nhd"), both
    cut from one tensor with a gap behind each row block ("mixed")."""
    el = torch.uint8 if dtype == E4M3 else torch.int16
    nan = 0x7F if dtype == E4M3 else 0x7FC0 if dtype == torch.bfloat16 else 0x7E00
    if layout == "hnd":
        k, v = (torch.full((pages, kv, page, hd), nan, dtype=el).view(dtype) for _ in range(2))
    elif layout == "nhd":
        k, v = (torch.full((pages, page, kv, hd), nan, dtype=el).view(dtype).transpose(1, 2) for _ in range(2))
    else:
        both = torch.full((pages, page, 2, kv, hd + 16), nan, dtype=el).view(dtype)
        k, v = (both[:, :, i, :, :hd].transpose(1, 2) for i in range(2))
    return k, v


def bits(t):
    return t.contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)


def put(pool, where, rows):
    """pool[page, :, slot] = rows, for 8-bit types too."""
    if pool.dtype == E4M3:
        for (page, slot), r in zip(where, rows):
            pool.view(torch.uint8)[page, :, slot] = r.view(torch.uint8)
    else:
        for (page, slot), r in zip(where, rows):
            pool[page, :, slot] = r


class Layer:
    """lens[b] positions for each sequence, the last rows[b] of them new. K and V are drawn in the cache's type (e4m3
    with scales); everything is on the CPU until dev()."""

    def __init__(self, seed, lens, rows, heads, kv, hd, page=16, qt="bf16", cache="same", layout="hnd", spare=0,
                 width=None, extra_pages=3):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.rows, self.heads, self.kv, self.hd, self.page = list(lens), list(rows), heads, kv, hd, page
        self.qt = QT[qt]
        self.ct = E4M3 if cache == "e4m3" else self.qt
        need = [-(-n // page) for n in lens]
        pages = sum(need) + extra_pages
        order = torch.randperm(pages, generator=g).tolist()
        width = width or max(max(need), 1) + 1
        self.table = torch.tensor([[2 ** 30 if i % 2 else -1 for i in range(width)] for _ in lens], dtype=torch.int32)
        self.kscale = self.vscale = None
        if cache == "e4m3":
            self.kscale = 0.01 + 0.01 * torch.rand(kv, generator=g)
            self.vscale = 0.005 + 0.01 * torch.rand(kv, generator=g)
        self.kpool, self.vpool = empty_pool(pages, kv, page, hd, self.ct, layout)
        self.K, self.V, self.where = [], [], []
        used = 0
        for b, n in enumerate(lens):
            mine = order[used:used + need[b]]
            used += need[b]
            self.table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
            self.where.append([(mine[p // page], p % page) for p in range(n)])
            for name, pool, scale in (("K", self.kpool, self.kscale), ("V", self.vpool, self.vscale)):
                x = torch.randn(n, kv, hd, generator=g)
                if scale is not None:
                    x = (x / scale[None, :, None]).clamp(-448, 448)
                x = x.to(self.ct)
                put(pool, self.where[b], x)
                x = x.double() if scale is None else x.double() * scale.double()[None, :, None]
                getattr(self, name).append(x)
        total = sum(rows) + spare
        self.q = (1.5 * torch.randn(total, heads * hd, generator=g)).to(self.qt)
        self.starts = torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32)
        self.lens_t = torch.tensor(lens, dtype=torch.int32)

    def dev(self, ops):
        """The pool's handle and the call's tensors on the GPU (the pool with its own strides)."""
        def up(t):
            d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
            i = torch.uint8 if t.dtype == E4M3 else None
            (d if i is None else d.view(i)).copy_(t if i is None else t.view(i))
            return d
        k, v = up(self.kpool), up(self.vpool)
        sc = [None if s is None else s.cuda() for s in (self.kscale, self.vscale)]
        return ops.PagedCache(k, v, *sc), self.q.cuda(), self.table.cuda(), self.lens_t.cuda(), self.starts.cuda()

    def want(self, y, decode=False, scale=None, window=0, sinks=0, hidden=()):
        """(y, what its values may be off by) in 64 bits, from the definition: rows that belong to no sequence as in
        `y`. hidden: (sequence, position) pairs that hold nothing."""
        scale = self.hd ** -0.5 if scale is None else scale
        out, tol = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
        group, hd = self.heads // self.kv, self.hd
        half_y, half_p = HALF[y.dtype], HALF[self.qt]
        first = 0
        for b, (n, r) in enumerate(zip(self.lens, self.rows)):
            for i in range(r):
                row, p = first + i, n - r + i
                j = torch.arange(n)
                see = (j <= p) & ((j > p - window) | (j < sinks) if window else torch.ones(n, dtype=torch.bool))
                for s, at in hidden:
                    if s == b:
                        see[at] = False
                j = j[see]
                if len(j) == 0:
                    out[row] = 0
                    continue
                K, V = (x[b][j].repeat_interleave(group, 1).transpose(0, 1) for x in (self.K, self.V))  # [heads, n, hd]
                q = self.q[row].double().view(self.heads, hd, 1)
                s = scale * (K @ q)[..., 0]
                w = torch.softmax(s, -1)
                o = (w[:, None, :] @ V)[:, 0]
                # Each numerator is rounded to q's type (half_p; in binary16 never finer than 2^-25 of the largest),
                # the scores are fp32 sums of hd products and the rest a few fp32 steps, counted for all the keys.
                ds = 2 * (hd + 8) * 2.0 ** -24 * scale * (K.abs() @ q.abs())[..., 0].amax(-1)
                rel = (half_p + 2 * ds + (16 + 2 * math.sqrt(len(j))) * 2.0 ** -24)[:, None]
                spread = (w[:, None, :] @ V.abs())[:, 0]
                t = rel * spread + half_y * (o.abs() + rel * spread)
                if self.qt == torch.float16:
                    t += 2.0 ** -25 * V.abs().sum(1) * w.amax(-1, keepdim=True)
                if y.dtype == torch.float16:
                    t += 2.0 ** -25
                out[row], tol[row] = o.reshape(-1), t.reshape(-1)
            first += r
        return out, tol


def compare(got, want, tol):
    got = got.cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), "not finite at %s" % (torch.nonzero(~torch.isfinite(got))[:4].tolist(),)
    far = (got - want).abs() - tol
    assert (far <= 0).all(), "off by %g more than %g at %s" % (far.max(), tol.reshape(-1)[far.argmax()],
                                                              divmod(int(far.argmax()), want.shape[1]))
