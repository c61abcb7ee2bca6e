"""Measured cases of a serving step's operators around the paged cache: projections in microscaled 4-bit floating point, the
norm and rotation of queries and keys on their way to attention, and the log probabilities that answer a request.

Kinds:
  product  ops.gemm_mx4: y = x w^T + bias, w in microscaled 4 bits; x a tensor that the call quantises, or in 4 bits already.
  pair     ops.quant_mx4 once, then two products of it (a gate and an up projection).
  rope     ops.qk_norm_rope: q and k rows, normed for each head and rotated by their positions.
  store    ops.kv_append_rope: the same, with the keys and the values going to their pages of a key / value cache.
  logprobs ops.token_logprobs: log probabilities of given tokens, the entropy and the top alternatives of rows of logits.

Microscaled 4 bits: blocks of 32 values of a row share a scale 2^(b - 127); b is the exponent field of the block's largest
magnitude in fp32, less 2 (0 at least). A value is x / scale rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (even code on
a tie, 6 past it) with x's sign. Codes are 4 bits, two to a byte, the even position in the low half.

Sequences are packed: rows starts[b] .. starts[b + 1] - 1 are the last positions of a sequence of lens[b]. Rows behind the last
sequence and idle slots (length 0) keep what their outputs held.

A row of logits that are all -infinity has entropy 0 and no probable token; a token outside the vocabulary has none either.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "mx4": 17 / 32}
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E4M3_MAX = 448.0
_EPS = 1e-6


def listed():
    return [
        # one token through a 0.6B decoder layer's query projection: latency
        {"name": "product_token", "kind": "product", "m": 1, "n": 2048, "k": 1024, "x": "bf16", "out": "bf16", "bias": False},
        # one token through that model's head: the weights' bytes
        {"name": "product_head", "kind": "product", "m": 1, "n": 151936, "k": 1024, "x": "bf16", "out": "fp32", "bias": False},
        # a decode batch of odd size through a wide up projection, with a bias
        {"name": "product_batch", "kind": "product", "m": 37, "n": 12288, "k": 1536, "x": "fp16", "out": "fp16", "bias": True},
        # a prompt's rows through gate and up, quantised once for both
        {"name": "pair_prompt", "kind": "pair", "m": 2011, "n": 12288, "k": 4096, "x": "bf16", "out": "bf16", "bias": False},
        # the largest product: a long prompt through a square projection, quantised by the step before
        {"name": "product_long", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "x": "mx4", "out": "bf16", "bias": False},
        # one token of one conversation, 16 / 8 heads of 128: latency
        {"name": "rope_token", "kind": "rope", "seqs": 1, "idle": 0, "past0": 1776, "past1": 1776, "rows0": 1, "rows1": 1,
         "spare": 0, "heads": 16, "kv_heads": 8, "hd": 128, "rot": 128, "q": "bf16", "norm": True, "plan": 1},
        # packed prompts of odd lengths, rows behind the last one
        {"name": "rope_prompts", "kind": "rope", "seqs": 7, "idle": 1, "past0": 0, "past1": 3000, "rows0": 200, "rows1": 2100,
         "spare": 37, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128, "q": "fp16", "norm": True, "plan": 2},
        # a decode batch with idle slots, keys and values into the cache
        {"name": "store_batch", "kind": "store", "seqs": 64, "idle": 3, "past0": 20, "past1": 8000, "rows0": 1, "rows1": 1,
         "spare": 0, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128, "q": "bf16", "norm": True, "page": 16, "cache": "bf16",
         "plan": 3},
        # chunks of long texts into an e4m3 cache, heads of 256 rotated over a quarter
        {"name": "store_prompts_e4m3", "kind": "store", "seqs": 6, "idle": 0, "past0": 1000, "past1": 9000, "rows0": 300,
         "rows1": 2050, "spare": 5, "heads": 8, "kv_heads": 4, "hd": 256, "rot": 64, "q": "bf16", "norm": True, "page": 64,
         "cache": "e4m3", "plan": 4},
        # one step's answer with five alternatives: latency
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": 151936, "x": "fp32", "given": 1, "top": 5,
         "masked": 0.0, "empty": 0},
        # a batch under grammars (most tokens masked, one row with nothing left), twenty alternatives
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 61, "vocab": 151936, "x": "bf16", "given": 2, "top": 20,
         "masked": 0.7, "empty": 1},
        # a prompt's tokens scored, with the most likely one beside each
        {"name": "logprobs_prompt", "kind": "logprobs", "rows": 2048, "vocab": 151936, "x": "bf16", "given": 1, "top": 1,
         "masked": 0.0, "empty": 0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def _draw_once(rng):
    kind = rng.choice(["product", "product", "pair", "rope", "store", "logprobs", "logprobs"])
    if kind in ("product", "pair"):
        x = rng.choice(["bf16", "fp16", "fp32", "mx4"] if kind == "product" else ["bf16", "fp16", "fp32"])
        out = rng.choice(["bf16", "fp32", "fp16"]) if x == "mx4" else x
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": _log(rng, 1, 151936), "k": 32 * _log(rng, 1, 512), "x": x, "out": out,
                "bias": kind == "product" and rng.random() < 0.4}
    if kind == "logprobs":
        return {"kind": kind, "rows": _log(rng, 1, 4096), "vocab": _log(rng, 1000, 262144), "x": rng.choice(["bf16", "fp16", "fp32"]),
                "given": rng.randrange(1, 5), "top": rng.choice([0, 1, 3, 10, 20, 64]), "masked": rng.choice([0.0, 0.0, 0.3, 0.95]),
                "empty": rng.choice([0, 0, 1])}
    kv_heads = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128, 256])
    case = {"kind": kind, "heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads, "hd": hd,
            "rot": rng.choice([hd, hd, hd // 2, hd // 4]), "q": rng.choice(["bf16", "fp16"]), "norm": rng.random() < 0.75,
            "plan": rng.randrange(1, 1 << 30)}
    if rng.random() < 0.5:
        case |= {"seqs": _log(rng, 1, 200), "past1": _log(rng, 1, 131072), "rows0": 1, "rows1": 1, "spare": 0}
    else:
        case |= {"seqs": _log(rng, 1, 24), "past1": rng.choice([0, _log(rng, 1, 16384)]), "rows1": _log(rng, 1, 8192),
                 "spare": rng.choice([0, 0, 1, 40])}
        case["rows0"] = rng.randrange(1, case["rows1"] + 1)
    case["past0"] = rng.randrange(0, case["past1"] + 1)
    case["idle"] = rng.randrange(0, 1 + case["seqs"] // 4)
    if kind == "store":
        case |= {"page": rng.choice([16, 32, 64, 128]), "cache": rng.choice([case["q"], case["q"], "e4m3"])}
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["bytes"] > 6e8 or w["flops"] > 1.1e12:
            continue
        if case["kind"] in ("product", "pair"):
            if case["m"] * case["n"] <= 1.2e8 and case["n"] * case["k"] <= 1.6e8:
                return case
        elif case["kind"] == "logprobs":
            if case["rows"] * case["vocab"] <= 3.1e8:
                return case
        else:
            lens, rows = _plan(case)
            if sum(lens) * case["kv_heads"] * case["hd"] <= 4e8 and sum(rows) <= 20000:
                return case


def _plan(case):
    """Each sequence's length (its new tokens included) and number of new tokens; the idle ones are among them."""
    rng = random.Random(case["plan"])
    lens, rows = [], []
    every = max(1, case["seqs"] // max(1, case["idle"]))
    for i in range(case["seqs"]):
        n = _log(rng, case["rows0"], case["rows1"])
        past = rng.randint(case["past0"], case["past1"])
        idle = i % every == every - 1 and lens.count(0) < case["idle"]
        lens.append(0 if idle else past + n)
        rows.append((1 if case["rows1"] == 1 else 0) if idle else n)
    return lens, rows


def work(case):
    if case["kind"] in ("product", "pair"):
        m, n, k, many = case["m"], case["n"], case["k"], 2 if case["kind"] == "pair" else 1
        return {"bytes": m * k * _SIZE[case["x"]] + many * (n * k * _SIZE["mx4"] + m * n * _SIZE[case["out"]]) + 4 * n * case["bias"],
                "flops": 2 * many * m * n * k}
    if case["kind"] == "logprobs":
        rows = case["rows"]
        return {"bytes": rows * (case["vocab"] * _SIZE[case["x"]] + 12 * case["given"] + 4 + 8 * case["top"]), "flops": 0}
    lens, rows = _plan(case)
    total = sum(r for n, r in zip(lens, rows) if n)
    positions = len({p for n, r in zip(lens, rows) for p in range(max(0, n - r), n)})
    heads, kv, hd = case["heads"], case["kv_heads"], case["hd"]
    meta = 4 * (2 * len(lens) + positions * case["rot"] + 2 * hd * case["norm"])
    if case["kind"] == "rope":
        return {"bytes": total * (heads + kv) * hd * 4 + meta, "flops": 0}
    el = 1 if case["cache"] == "e4m3" else 2
    return {"bytes": total * hd * (4 * heads + 2 * kv * (2 + el)) + meta + 4 * sum(-(-n // case["page"]) for n in lens), "flops": 0}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = dict(case)
    make = {"product": _make_product, "pair": _make_product, "rope": _make_rows, "store": _make_rows, "logprobs": _make_logits}
    make[case["kind"]](case, state, g)
    return state


def _make_codes(g, rows, cols):
    """A matrix as its quantisation leaves it: codes, and scales of a few neighbouring powers of two."""
    codes = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    spread = torch.randint(0, 4, (rows, cols // 32), generator=g, device="cuda", dtype=torch.uint8)
    return codes, spread + 119


def _make_product(case, state, g):
    m, n, k = case["m"], case["n"], case["k"]
    state["w"] = [_make_codes(g, n, k) for _ in range(2 if case["kind"] == "pair" else 1)]
    if case["x"] == "mx4":
        state["mx"] = _make_codes(g, m, k)
    else:  # activations: a few columns far above the others, an all-zero row (padding) in a batch
        x = torch.randn(m, k, generator=g, device="cuda")
        x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.02, 12.0, 1.0)
        if m > 4:
            x[m // 3] = 0
        state["tensor"] = x.to(_T[case["x"]])
    state["b"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    if own:  # the handles that a program makes once, when it loads its weights
        from opentars_amd import ops
        state["own_w"] = [ops.Mx4(*w) for w in state["w"]]
        if case["x"] == "mx4":
            state["own_x"] = ops.Mx4(*state["mx"])


def _make_rows(case, state, g):
    lens, rows = _plan(case)
    t, heads, kv, hd = _T[case["q"]], case["heads"], case["kv_heads"], case["hd"]
    total = sum(rows) + case["spare"]
    fused = torch.randn(total, (heads + 2 * kv) * hd, generator=g, device="cuda", dtype=t)  # one projection's q, k and v
    state["q_rows"], state["k_rows"], state["v_rows"] = fused.split([heads * hd, kv * hd, kv * hd], 1)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    decode = case["rows1"] == 1
    state["starts"] = None if decode else torch.cumsum(torch.tensor([0] + rows, device="cuda"), 0).to(torch.int32)
    state["qg"] = state["kg"] = None
    if case["norm"]:
        state["qg"], state["kg"] = 1 + 0.2 * torch.randn(2, hd, generator=g, device="cuda")
    half = case["rot"] // 2
    angle = torch.arange(max(lens) + 1, dtype=torch.float64, device="cuda")[:, None] * 1e6 ** (
        -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    state["tab"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    state["yq"] = torch.randn(total, heads * hd, generator=g, device="cuda", dtype=t)
    if case["kind"] == "rope":
        state["yk"] = torch.randn(total, kv * hd, generator=g, device="cuda", dtype=t)
        return
    page = case["page"]
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 3, max(max(need), 1) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    n_t = torch.tensor(need, device="cuda")
    first, col = torch.cumsum(n_t, 0) - n_t, torch.arange(width, device="cuda")
    state["table"] = torch.where(col < n_t[:, None], order[(first[:, None] + col).clamp(max=pages - 1)], -1).to(torch.int32)
    kc, vc, state["scales"] = *torch.randn(2, pages, kv, page, hd, generator=g, device="cuda", dtype=t), None
    if case["cache"] == "e4m3":
        state["scales"] = 0.008 + 0.004 * torch.rand(2, kv, generator=g, device="cuda")
        kc, vc = ((c * 80).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn) for c in (kc, vc))
    state["kc"], state["vc"] = kc, vc
    if own:  # the cache's handle, made once with its pool
        from opentars_amd import ops
        state["handle"] = ops.PagedCache(kc, vc) if state["scales"] is None else ops.PagedCache(kc, vc, *state["scales"])


def _make_logits(case, state, g):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn(rows, vocab, generator=g, device="cuda", dtype=_T[case["x"]])
    x *= 2.5
    peak = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")  # what a trained head is sure of
    x.scatter_add_(1, peak, (4 + 8 * torch.rand(rows, 8, generator=g, device="cuda")).to(x.dtype))
    if case["masked"]:
        x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"], -math.inf)
    if case["empty"]:
        x[rows // 2] = -math.inf
    tokens = torch.randint(0, vocab, (rows, case["given"]), generator=g, device="cuda")
    tokens[:, 0] = peak[:, 0]
    if rows > 8:
        tokens[rows - 2:] = -1  # a padded batch
    state["logits"], state["tokens"] = x, tokens


def run(state):
    kind = state["kind"]
    if own:
        from opentars_amd import ops
        if kind == "product":
            x = state["own_x"] if state["x"] == "mx4" else state["tensor"]
            out = {"bf16": ops.OUT_BF16, "fp16": ops.OUT_FP16, "fp32": ops.OUT_FP32}[state["out"]]
            return {"y": ops.gemm_mx4(x, state["own_w"][0], bias=state["b"], out=out)}
        if kind == "pair":
            x = ops.quant_mx4(state["tensor"])
            out = {"bf16": ops.OUT_BF16, "fp16": ops.OUT_FP16, "fp32": ops.OUT_FP32}[state["out"]]
            return {"gate": ops.gemm_mx4(x, state["own_w"][0], out=out), "up": ops.gemm_mx4(x, state["own_w"][1], out=out)}
        if kind == "rope":
            q, k = ops.qk_norm_rope(state["q_rows"], state["k_rows"], state["hd"], state["tab"], state["lens"], state["starts"],
                                    qgamma=state["qg"], kgamma=state["kg"], eps=_EPS, yq=state["yq"], yk=state["yk"])
            return {"q": q, "k": k}
        if kind == "store":
            q = ops.kv_append_rope(state["handle"], state["q_rows"], state["k_rows"], state["v_rows"], state["table"], state["lens"],
                                   state["tab"], state["starts"], qgamma=state["qg"], kgamma=state["kg"], eps=_EPS, yq=state["yq"])
            return {"q": q, "k": state["kc"], "v": state["vc"]}
        r = ops.token_logprobs(state["logits"], state["tokens"], top=state["top"])
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top": r.top_logprobs, "ids": r.top_ids}
    if kind == "product":
        x = _values(*state["mx"]) if state["x"] == "mx4" else _quantised(state["tensor"])
        y = torch.matmul(x, _values(*state["w"][0]).t())
        if state["b"] is not None:
            y += state["b"]
        return {"y": y.to(_T[state["out"]])}
    if kind == "pair":
        x = _quantised(state["tensor"])
        gate, up = (torch.matmul(x, _values(*w).t()).to(_T[state["out"]]) for w in state["w"])
        return {"gate": gate, "up": up}
    if kind == "rope":
        row, _, pos = _where(state)
        yq, yk = state["yq"].clone(), state["yk"].clone()
        yq[row] = _rotated(state, "q_rows", "qg", row, pos).flatten(1).to(yq.dtype)
        yk[row] = _rotated(state, "k_rows", "kg", row, pos).flatten(1).to(yk.dtype)
        return {"q": yq, "k": yk}
    return _store(state) if kind == "store" else _logprobs(state)


def _power(b):
    """2^(b - 127) for scale bytes b below 255."""
    return torch.where(b > 0, b.int() << 23, 1 << 22).view(torch.float32)


def _values(codes, scales):
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1, 32)
    return (grid[c.int()] * _power(scales)[..., None]).flatten(1)


def _quantised(x):
    """The values that x's codes and scales stand for."""
    x = x.float().view(x.shape[0], -1, 32)
    b = ((x.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=0)
    inv = ((254 - b) << 23).view(torch.float32)
    a = (x * inv[..., None]).abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    v = torch.tensor(_GRID, device=x.device)[code] * _power(b)[..., None]
    return torch.copysign(v, x).flatten(1)


def _where(state):
    """For every row that has a position: row, sequence, position."""
    lens = state["lens"].long()
    row = torch.arange(state["q_rows"].shape[0], device=lens.device)
    if state["starts"] is None:
        seq, pos = row, lens - 1
        here = pos >= 0
    else:
        starts = state["starts"].long()
        seq = torch.searchsorted(starts[1:], row, right=True)
        here = seq < lens.numel()
        seq = seq.clamp(max=lens.numel() - 1)
        pos = lens[seq] - starts[seq + 1] + row
        here &= pos >= 0
    return row[here], seq[here], pos[here]


def _rotated(state, name, gamma, row, pos):
    """[rows, heads, hd] in fp32."""
    hd, half = state["hd"], state["rot"] // 2
    x = state[name][row].float().view(len(row), -1, hd)
    if state[gamma] is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * state[gamma]
    c, s = state["tab"][pos][:, None].split(half, 2)
    a, b, rest = x.split([half, half, hd - 2 * half], 2)
    return torch.cat([a * c - b * s, b * c + a * s, rest], 2)


def _store(state):
    row, seq, pos = _where(state)
    yq = state["yq"].clone()
    yq[row] = _rotated(state, "q_rows", "qg", row, pos).flatten(1).to(yq.dtype)
    page = state["page"]
    at = state["table"][seq, pos // page].long()
    k = _rotated(state, "k_rows", "kg", row, pos)
    v = state["v_rows"][row].float().view(k.shape)
    for i, (x, cache) in enumerate(((k, state["kc"]), (v, state["vc"]))):
        if state["scales"] is not None:
            x = (x / state["scales"][i].view(1, -1, 1)).clamp(-_E4M3_MAX, _E4M3_MAX).to(cache.dtype).view(torch.uint8)
            cache = cache.view(torch.uint8)
        cache[at, :, pos % page] = x.to(cache.dtype)
    return {"q": yq, "k": state["kc"], "v": state["vc"]}


def _logprobs(state):
    x, tokens, top = state["logits"].float(), state["tokens"], state["top"]
    vocab = x.shape[1]
    most = x.amax(1, keepdim=True)
    none = most == -math.inf
    d = x - most.masked_fill(none, 0.0)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log = total.masked_fill(none, 1.0).log()
    entropy = log - d.masked_fill(d == -math.inf, 0.0).mul_(e).sum(1, keepdim=True) / total.masked_fill(none, 1.0)
    base = most.masked_fill(none, 0.0) + log
    inside = (tokens >= 0) & (tokens < vocab)
    given = torch.where(inside, x.gather(1, tokens.clamp(0, vocab - 1)) - base, -math.inf)
    if not top:
        return {"logprobs": given, "entropy": entropy[:, 0], "top": None, "ids": None}
    # whole-number keys that no two places share: the value's order above the place's, counted down
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long().mul_(1 << 32).add_(vocab - 1 - torch.arange(vocab, device=x.device))
    ids = vocab - 1 - (key.topk(top, 1).values & 0xFFFFFFFF)
    return {"logprobs": given, "entropy": entropy[:, 0], "top": x.gather(1, ids) - base, "ids": ids.int()}


def exact(case, seed):
    state = prepare(case, seed)
    return {"product": _exact_product, "pair": _exact_product, "rope": _exact_rows, "store": _exact_rows, "logprobs": _exact_logits}[
        case["kind"]](case, state)


def _exact_matrix(codes, scales):
    grid = torch.tensor([s * v for s in (1, -1) for v in _GRID], dtype=torch.float64, device=codes.device)
    v = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    v[:, 0::2], v[:, 1::2] = grid[(codes % 16).long()], grid[(codes // 16).long()]
    return v * torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, 1)


def _exact_quantised(x):
    d = x.double().view(-1, 32)
    largest = d.abs().amax(1, keepdim=True)
    exponent = torch.where(largest > 0, torch.frexp(largest).exponent - 3, -127).clamp(min=-127)
    scale = torch.ldexp(torch.ones_like(largest), exponent)
    q = (d / scale).abs()
    step = torch.where(q < 2, 0.5, torch.where(q < 4, 1.0, 2.0))
    q = (torch.round(q / step) * step).clamp(max=6.0)  # each binade's steps; round() takes ties to even
    return (q * d.sign() * scale).view(x.shape)


def _exact_product(case, state):
    x = _exact_matrix(*state["mx"]) if case["x"] == "mx4" else _exact_quantised(state["tensor"])
    ys = []
    for w in state["w"]:
        y = x @ _exact_matrix(*w).T
        ys.append(y if state["b"] is None else y + state["b"].double())
    return {"y": ys[0]} if case["kind"] == "product" else {"gate": ys[0], "up": ys[1]}


def _exact_rows(case, state):
    lens, rows = _plan(case)
    hd, half, d = case["hd"], case["rot"] // 2, torch.float64
    out = {"q": state["yq"].to(d)}
    if case["kind"] == "rope":
        out["k"] = state["yk"].to(d)
    else:
        out["k"], out["v"] = state["kc"].to(d), state["vc"].to(d)
    first = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        if n:
            p = torch.arange(n - r, n, device="cuda")
            done = {}
            for name, rows_of, gamma in (("q", "q_rows", "qg"), ("k", "k_rows", "kg")):
                x = state[rows_of][first:first + r].to(d).unflatten(1, (-1, hd))
                if case["norm"]:
                    x = x * (x.square().mean(2, keepdim=True) + _EPS).rsqrt() * state[gamma].to(d)
                t = state["tab"][n - r:n].to(d)
                z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(t[:, :half], t[:, half:])[:, None]
                done[name] = torch.cat([z.real, z.imag, x[..., 2 * half:]], 2)
            out["q"][first:first + r] = done["q"].flatten(1)
            if case["kind"] == "rope":
                out["k"][first:first + r] = done["k"].flatten(1)
            else:
                done["v"] = state["v_rows"][first:first + r].to(d).unflatten(1, (-1, hd))
                for i, name in enumerate("kv"):
                    x = done[name]
                    if state["scales"] is not None:
                        x = (x / state["scales"][i].to(d)[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
                    out[name][state["table"][b].long()[p // case["page"]], :, p % case["page"]] = x
        first += r
    return out


def _exact_logits(case, state):
    got = {"logprobs": [], "entropy": [], "top": [], "ids": []}
    for x, tokens in zip(state["logits"].split(256), state["tokens"].split(256)):
        x = x.double()
        none = (x == -math.inf).all(1, keepdim=True)
        lp = torch.log_softmax(x, 1).masked_fill(none, -math.inf)
        entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
        valid = (tokens >= 0) & (tokens < case["vocab"])
        got["logprobs"].append(lp.gather(1, tokens * valid).masked_fill(~valid, -math.inf))
        got["entropy"].append(entropy)
        if case["top"]:
            order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case["top"]]
            got["ids"].append(order.int())
            got["top"].append(lp.gather(1, order))
    return {name: torch.cat(v) if v else None for name, v in got.items()}
