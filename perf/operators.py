"""Measured cases of the paged key / value cache: storing new tokens in it, and the two attentions that read it.

Kinds:
  append  ops.kv_append: the K and V rows of new tokens go to their pages (as they are, or as e4m3 values with a
          scale for each K / V head).
  decode  ops.paged_decode: one query row per sequence over that sequence's whole cache.
  prompt  ops.paged_attention: the query rows of a prompt (a chunk of it, or a speculative round's few rows) over
          the cache that already holds them: causal, sequences packed one after another.

A sequence of length len holds positions 0 .. len - 1 in the pages its table row names, `page` positions a page.
Its `rows` new tokens are the last of them. With a window w and s sinks, the row at position p sees the positions
j <= p with j > p - w or j < s. y = softmax(scale q K^T) V over what the row sees; a row that sees nothing is zero,
and the rows behind the last sequence stay as they were.

A case's lengths are drawn from its own "plan" number, so that its work is the same for every seed of its data.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_Q = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3_MAX = 448.0


def listed():
    return [
        # one new token of one conversation (16 query / 8 K / V heads of 128, as a 0.6B decoder layer): latency
        {"name": "append_token", "kind": "append", "seqs": 1, "idle": 0, "past0": 1776, "past1": 1776, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 16, "kv_heads": 8, "hd": 128, "page": 16, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 1},
        # the new tokens of a batch of prompt chunks, odd lengths, into an e4m3 cache
        {"name": "append_prompts_e4m3", "kind": "append", "seqs": 9, "idle": 1, "past0": 0, "past1": 5000,
         "rows0": 100, "rows1": 2100, "spare": 37, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "q": "bf16",
         "cache": "e4m3", "window": 0, "sinks": 0, "plan": 2},
        # one conversation, one token: a short cache, latency
        {"name": "decode_one", "kind": "decode", "seqs": 1, "idle": 0, "past0": 2046, "past1": 2046, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 16, "kv_heads": 8, "hd": 128, "page": 16, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 3},
        # a serving batch: 64 slots of very different lengths, three of them idle
        {"name": "decode_batch", "kind": "decode", "seqs": 64, "idle": 3, "past0": 20, "past1": 8000, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 4},
        # a few long documents: the cache's length is all there is to split
        {"name": "decode_long", "kind": "decode", "seqs": 3, "idle": 0, "past0": 90000, "past1": 131000, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 5},
        # many query heads for each K / V head over an e4m3 cache
        {"name": "decode_e4m3", "kind": "decode", "seqs": 32, "idle": 0, "past0": 9000, "past1": 17000, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 64, "kv_heads": 8, "hd": 128, "page": 32, "q": "bf16", "cache": "e4m3",
         "window": 0, "sinks": 0, "plan": 6},
        # a sliding layer (4 query heads over one K / V head of 256, window 512) far into its texts, binary16
        {"name": "decode_window", "kind": "decode", "seqs": 100, "idle": 0, "past0": 300, "past1": 30000, "rows0": 1,
         "rows1": 1, "spare": 0, "heads": 4, "kv_heads": 1, "hd": 256, "page": 16, "q": "fp16", "cache": "fp16",
         "window": 512, "sinks": 4, "plan": 7},
        # a short question after a short text, heads of 64: latency
        {"name": "prompt_short", "kind": "prompt", "seqs": 1, "idle": 0, "past0": 300, "past1": 300, "rows0": 77,
         "rows1": 77, "spare": 0, "heads": 16, "kv_heads": 4, "hd": 64, "page": 16, "q": "fp16", "cache": "fp16",
         "window": 0, "sinks": 0, "plan": 8},
        # speculative rounds: five rows for each sequence over long caches
        {"name": "prompt_rounds", "kind": "prompt", "seqs": 16, "idle": 0, "past0": 3000, "past1": 16000, "rows0": 5,
         "rows1": 5, "spare": 0, "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 9},
        # a batch of prompts of very different lengths, some with a cached prefix, rows behind the last one
        {"name": "prompt_batch", "kind": "prompt", "seqs": 11, "idle": 1, "past0": 0, "past1": 1500, "rows0": 60,
         "rows1": 2000, "spare": 29, "heads": 32, "kv_heads": 8, "hd": 128, "page": 16, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 10},
        # one long prompt: the largest product
        {"name": "prompt_long", "kind": "prompt", "seqs": 1, "idle": 0, "past0": 0, "past1": 0, "rows0": 8192,
         "rows1": 8192, "spare": 0, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64, "q": "bf16", "cache": "bf16",
         "window": 0, "sinks": 0, "plan": 11},
        # a chunk of a long text through a sliding layer with heads of 256, e4m3 cache
        {"name": "prompt_window_e4m3", "kind": "prompt", "seqs": 2, "idle": 0, "past0": 5000, "past1": 9000,
         "rows0": 2000, "rows1": 3001, "spare": 0, "heads": 8, "kv_heads": 4, "hd": 256, "page": 32, "q": "bf16",
         "cache": "e4m3", "window": 1024, "sinks": 4, "plan": 12},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def _draw_once(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    case = {"kind": kind, "heads": kv_heads * group, "kv_heads": kv_heads, "hd": rng.choice([64, 128, 128, 256]),
            "page": rng.choice([16, 32, 64, 128]), "q": rng.choice(["bf16", "fp16"]), "window": 0, "sinks": 0,
            "plan": rng.randrange(1, 1 << 30), "idle": 0, "spare": 0}
    case["cache"] = rng.choice([case["q"], case["q"], "e4m3"])
    if kind != "append" and rng.random() < 0.4:
        case["window"] = _log(rng, 16, 4096)
        case["sinks"] = rng.choice([0, 1, 4, 16, 70])
    if kind == "decode":
        case["seqs"] = _log(rng, 1, 200)
        case["past1"] = _log(rng, 1, 131072)
        case["past0"] = rng.randrange(0, case["past1"] + 1)
        case["rows0"] = case["rows1"] = 1
        case["idle"] = rng.randrange(0, 1 + case["seqs"] // 4)
    else:
        case["seqs"] = _log(rng, 1, 24)
        case["past1"] = rng.choice([0, _log(rng, 1, 16384)])
        case["past0"] = rng.randrange(0, case["past1"] + 1)
        case["rows1"] = _log(rng, 1, 8192)
        case["rows0"] = rng.randrange(1, case["rows1"] + 1)
        case["idle"] = rng.randrange(0, 1 + case["seqs"] // 4)
        case["spare"] = rng.choice([0, 0, 1, 40])
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        lens, rows = _plan(case)
        pool = sum(lens) * case["kv_heads"] * case["hd"]
        scores = len(lens) * case["heads"] * max(rows) * max(lens)
        if w["bytes"] <= 1.4e9 and w["flops"] <= 5.4e11 and pool <= 4e8 and scores <= 2.2e9 and sum(rows) <= 20000:
            return case


def _plan(case):
    """Each sequence's length (its new tokens included) and number of new tokens; the idle ones are among them."""
    rng = random.Random(case["plan"])
    lens, rows = [], []
    for i in range(case["seqs"]):
        n = _log(rng, case["rows0"], case["rows1"])
        past = rng.randint(case["past0"], case["past1"])
        idle = i % max(1, case["seqs"] // max(1, case["idle"])) == 1 and len([r for r in lens if r == 0]) < case["idle"]
        if idle:  # a decode batch keeps the slot's row, a packed batch has no row for it
            lens.append(0)
            rows.append(1 if case["kind"] == "decode" else 0)
        else:
            lens.append(past + n)
            rows.append(n)
    return lens, rows


def _visible(case, lens, rows):
    """Pairs of a row and a position it sees, and positions that some row of their sequence sees."""
    w, s, pairs, seen = case["window"], case["sinks"], 0, 0
    for n, r in zip(lens, rows):
        if n < r:
            continue
        if not w:
            pairs += r * (n - r) + r * (r + 1) // 2
            seen += n
            continue
        for p in range(n - r, n):
            pairs += min(p + 1, w) + min(s, max(0, p + 1 - w))
        lo = max(0, n - r + 1 - w)
        seen += n - lo + min(s, lo)
    return pairs, seen


def work(case):
    lens, rows = _plan(case)
    el = 1 if case["cache"] == "e4m3" else 2
    total, kv = sum(r for n, r in zip(lens, rows) if n), case["kv_heads"] * case["hd"]
    meta = 4 * (len(lens) * 2 + sum(-(-n // case["page"]) for n in lens))
    if case["kind"] == "append":
        return {"bytes": total * kv * 2 * (2 + el) + meta, "flops": 0}
    pairs, seen = _visible(case, lens, rows)
    return {"bytes": seen * kv * 2 * el + total * case["heads"] * case["hd"] * 4 + meta,
            "flops": 4 * pairs * case["heads"] * case["hd"]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lens, rows = _plan(case)
    qt, kv, hd, page, heads = _Q[case["q"]], case["kv_heads"], case["hd"], case["page"], case["heads"]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    width = max(max(need), 1) + 1
    # the pool's pages go to the sequences in no order; a table row ends in entries that name no page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    n_t = torch.tensor(need, device="cuda")
    first = torch.cumsum(n_t, 0) - n_t
    col = torch.arange(width, device="cuda")
    table = torch.where(col < n_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).to(torch.int32)
    total = sum(rows) + case["spare"]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=qt)  # noqa: E731
    kc, vc, scales = randn(pages, kv, page, hd), randn(pages, kv, page, hd), None
    if case["cache"] == "e4m3":  # scales that put four or so standard deviations at e4m3's end
        scales = (0.008 + 0.004 * torch.rand(2, kv, generator=g, device="cuda"))
        kc = (kc / scales[0].view(1, kv, 1, 1).to(qt)).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
        vc = (vc / scales[1].view(1, kv, 1, 1).to(qt)).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    ends = torch.cumsum(torch.tensor([0] + rows, device="cuda"), 0).to(torch.int32)
    state = {"kind": case["kind"], "kc": kc, "vc": vc, "scales": scales, "table": table, "window": case["window"],
             "sinks": case["sinks"], "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "heads": heads,
             "starts": ends, "most": (max(lens), max(rows))}
    if case["kind"] == "append":
        state["k"], state["v"] = randn(total, kv * hd), randn(total, kv * hd)
    else:
        state["q"], state["y"] = 2.0 * randn(total, heads * hd), randn(total, heads * hd)
    if own:  # the handle of the cache that a program makes once, with its pool
        from opentars_amd import ops
        state["cache"] = ops.PagedCache(kc, vc) if scales is None else ops.PagedCache(kc, vc, scales[0], scales[1])
    return state


def run(state):
    kind = state["kind"]
    if own:
        from opentars_amd import ops
        if kind == "append":
            ops.kv_append(state["cache"], state["k"], state["v"], state["table"], state["lens"], state["starts"])
            return {"k": state["kc"], "v": state["vc"]}
        if kind == "decode":
            return {"y": ops.paged_decode(state["cache"], state["q"], state["table"], state["lens"],
                                          window=state["window"], sinks=state["sinks"], y=state["y"])}
        return {"y": ops.paged_attention(state["cache"], state["q"], state["table"], state["lens"], state["starts"],
                                         window=state["window"], sinks=state["sinks"], y=state["y"])}
    return _append(state) if kind == "append" else _attend(state)


def _where(state):
    """For every row that belongs to a sequence and has a position: row, sequence, position."""
    starts, lens = state["starts"].long(), state["lens"].long()
    row = torch.arange(state["k" if state["kind"] == "append" else "q"].shape[0], device=starts.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    here = seq < lens.numel()
    seq = seq.clamp(max=lens.numel() - 1)
    pos = lens[seq] - starts[seq + 1] + row
    here &= pos >= 0
    return row[here], seq[here], pos[here]


def _append(state):
    row, seq, pos = _where(state)
    kc, vc = state["kc"], state["vc"]
    kv, page, hd = kc.shape[1:]
    at = state["table"][seq, pos // page].long()
    for name, cache in (("k", kc), ("v", vc)):
        x = state[name][row].view(-1, kv, hd)
        if state["scales"] is not None:
            x = x.float() / state["scales"][0 if name == "k" else 1].view(1, kv, 1)
            x = x.clamp(-_E4M3_MAX, _E4M3_MAX).to(cache.dtype).view(torch.uint8)
            cache = cache.view(torch.uint8)
        cache[at, :, pos % page] = x
    return {"k": kc, "v": vc}


def _attend(state):
    q, kc, vc, lens, starts = state["q"], state["kc"], state["vc"], state["lens"].long(), state["starts"].long()
    kv, page, hd = kc.shape[1:]
    seqs, group, (longest, most) = lens.numel(), state["heads"] // kv, state["most"]
    pos = torch.arange(longest, device=q.device)
    at = state["table"][:, pos // page].long().clamp(min=0)
    here = (pos < lens[:, None])[:, None, None, :]

    def gathered(cache, scale):
        if scale is None:
            return cache[at, :, pos % page].float().transpose(1, 2).contiguous()          # [seqs, kv, longest, hd]
        x = cache.view(torch.uint8)[at, :, pos % page].view(cache.dtype).float() * scale.view(1, 1, kv, 1)
        return x.transpose(1, 2).contiguous()

    scales = (None, None) if state["scales"] is None else state["scales"]
    new = torch.arange(most, device=q.device)
    row = (starts[:-1, None] + new).clamp(max=q.shape[0] - 1)
    mine = new < (starts[1:] - starts[:-1])[:, None]
    x = q[row].float().view(seqs, most, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, hd)
    s = torch.matmul(x, gathered(kc, scales[0]).transpose(2, 3)).view(seqs, kv * group, most, longest)
    s *= 1.0 / math.sqrt(hd)
    p = (lens[:, None] - (starts[1:] - starts[:-1])[:, None] + new)[:, None, :, None]    # the rows' positions
    sees = here & (pos <= p)
    if state["window"]:
        sees = sees & ((pos > p - state["window"]) | (pos < state["sinks"]))
    s.masked_fill_(~sees, -math.inf)
    top = s.amax(-1, keepdim=True)
    s = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    s = s.div_(total.masked_fill(total == 0, 1.0)).view(seqs, kv, group * most, longest)
    o = torch.matmul(s, gathered(vc, scales[1]).masked_fill((pos >= lens[:, None])[:, None, :, None], 0.0))
    o = o.view(seqs, kv, group, most, hd).permute(0, 3, 1, 2, 4).reshape(seqs, most, kv * group * hd)
    y = state["y"].clone()
    y[row[mine]] = o[mine].to(y.dtype)
    return {"y": y}


def exact(case, seed):
    state = prepare(case, seed)
    lens, rows = _plan(case)
    kv, hd, page, group = case["kv_heads"], case["hd"], case["page"], case["heads"] // case["kv_heads"]
    scale = [None if state["scales"] is None else t.double() for t in (state["scales"] if state["scales"] is not None else (0, 0))]
    d = torch.float64
    if case["kind"] == "append":
        out = {"k": state["kc"].to(d), "v": state["vc"].to(d)}
        for j, name in enumerate("kv"):
            first = 0
            for b, (n, r) in enumerate(zip(lens, rows)):
                for h in range(kv):
                    x = state[name][first:first + r, h * hd:(h + 1) * hd].to(d)
                    if scale[j] is not None:
                        x = (x / scale[j][h]).clamp(-_E4M3_MAX, _E4M3_MAX)
                    p = torch.arange(n - r, n, device=x.device)
                    out[name][state["table"][b].long()[p // page], h, p % page] = x
                first += r
        return out
    y = state["y"].to(d)
    first = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        if n == 0:
            y[first:first + r] = 0
        else:
            j = torch.arange(n, device=y.device)
            pages = state["table"][b, :-(-n // page)].long()
            p = torch.arange(n - r, n, device=y.device)
            dark = j[None, :] > p[:, None]
            if case["window"]:
                dark |= (j[None, :] <= p[:, None] - case["window"]) & (j[None, :] >= case["sinks"])
            for h in range(kv):
                K, V = ((c[pages, h].to(d).reshape(-1, hd)[:n]) for c in (state["kc"], state["vc"]))
                if scale[0] is not None:
                    K, V = K * scale[0][h], V * scale[1][h]
                for i in range(h * group, (h + 1) * group):
                    cols = slice(i * hd, (i + 1) * hd)
                    t = state["q"][first:first + r, cols].to(d) @ K.T / math.sqrt(hd)
                    y[first:first + r, cols] = torch.softmax(t.masked_fill_(dark, -math.inf), -1) @ V
        first += r
    return {"y": y}
