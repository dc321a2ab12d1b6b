"""Cases of the sequence operators: attention over packed sequences, the 8-bit paged key / value cache
(append, read back, single-token attention) and the logit rules.

Run as a module by a timing harness: `listed()` and `draw(rng)` give cases, `prepare(case, seed)` what a program
holds before the call, `run(state)` one pass, `work(case)` the bytes and operations that pass cannot do without,
`exact(case, seed)` the same outputs in 64 bits.  With `own` false `run` computes the operators from elementary
torch operations; with `own` true it calls ppocr_b200.
"""

import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_handle = None


def _gpu():
    """The framework's device handle, made once per process as a program does."""
    global _handle
    if _handle is None:
        path = os.path.join(_ROOT, "ppocr-rs_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import ppocr_b200 as P

        _handle = (P, P.Gpu(torch.cuda.current_device()))
    return _handle


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The medium recognizer's encoder over 256 text lines of different widths (8 heads of 24, up to 160 steps),
        # packed without the padding of a common canvas.
        {"name": "lines bf16", "op": "attention_packed", "dtype": "bf16", "sequences": 256, "shortest": 20,
         "longest": 160, "heads": 8, "kv_heads": 8, "d": 24, "causal": False, "keys": "same"},
        # The small recognizer's heads (8 of 15) in the FP32 mode, a page's worth of lines.
        {"name": "lines f32", "op": "attention_packed", "dtype": "f32", "sequences": 64, "shortest": 4,
         "longest": 200, "heads": 8, "kv_heads": 8, "d": 15, "causal": False, "keys": "same"},
        # Prompts of several requests in one pass, ragged, grouped heads.
        {"name": "prompts bf16", "op": "attention_packed", "dtype": "bf16", "sequences": 7, "shortest": 1,
         "longest": 2500, "heads": 32, "kv_heads": 8, "d": 128, "causal": True, "keys": "same"},
        # One long prompt, an odd length.
        {"name": "long prompt bf16", "op": "attention_packed", "dtype": "bf16", "sequences": 1, "shortest": 8191,
         "longest": 8191, "heads": 16, "kv_heads": 2, "d": 128, "causal": True, "keys": "same"},
        # A few requests' next chunk behind what they hold already (more keys than queries), FP32.
        {"name": "chunks f32", "op": "attention_packed", "dtype": "f32", "sequences": 3, "shortest": 64,
         "longest": 700, "heads": 16, "kv_heads": 4, "d": 64, "causal": True, "keys": "more"},
        # One request early in its answer: the latency of a single step.
        {"name": "step alone bf16", "op": "attention_cached", "dtype": "bf16", "sequences": 1, "shortest": 101,
         "longest": 101, "heads": 8, "kv_heads": 2, "d": 64, "page": 16},
        # A serving batch in the middle of its answers.
        {"name": "step batch bf16", "op": "attention_cached", "dtype": "bf16", "sequences": 64, "shortest": 1,
         "longest": 4100, "heads": 32, "kv_heads": 8, "d": 128, "page": 32},
        # Two requests over long contexts, FP32.
        {"name": "step long f32", "op": "attention_cached", "dtype": "f32", "sequences": 2, "shortest": 30000,
         "longest": 65000, "heads": 24, "kv_heads": 8, "d": 128, "page": 64},
        # Prompts written into the cache in one call, then read back as the values the cache holds.
        {"name": "append prompts bf16", "op": "cache_append", "dtype": "bf16", "sequences": 8, "shortest": 33,
         "longest": 2000, "held": 0, "kv_heads": 8, "d": 128, "page": 32},
        # One new token for each request of a large batch: partly filled blocks whose scale may grow.
        {"name": "append tokens f32", "op": "cache_append", "dtype": "f32", "sequences": 256, "shortest": 1,
         "longest": 1, "held": 900, "kv_heads": 4, "d": 64, "page": 16},
        # Every step of 256 lines of 40 steps through the tiny recognizer's classifier, held to one set of classes.
        {"name": "rules lines f32", "op": "logit_rules", "dtype": "f32", "rows": 10240, "vocab": 6906, "history": 0,
         "states": 1, "bias": True, "penalties": False},
        # One step of a serving batch: penalties over what each request has written, a bias, a grammar state per row.
        {"name": "rules batch bf16", "op": "logit_rules", "dtype": "bf16", "rows": 64, "vocab": 128000,
         "history": 4000, "states": 16, "bias": True, "penalties": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention_packed", "attention_packed", "attention_cached", "attention_cached", "cache_append",
                     "logit_rules"])
    dtype = rng.choice(["bf16", "f32"])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    if op == "attention_packed":
        d = rng.choice([8, 15, 16, 24, 32, 40, 64, 80, 96, 128, rng.randint(1, 128)])
        longest = _log(rng, 1, 4096)
        case = {"op": op, "dtype": dtype, "sequences": _log(rng, 1, 128), "shortest": rng.choice([0, 1, longest]),
                "longest": longest, "heads": heads, "kv_heads": kv, "d": d, "causal": rng.random() < 0.6,
                "keys": rng.choice(["same", "same", "more", "fewer"])}
        # What the padded plain form has to hold stays below the long prompt's.
        while case["sequences"] * heads * longest * longest * (4 if case["keys"] == "more" else 1) > 4e8:
            case["sequences"] = max(1, case["sequences"] // 2)
            if case["sequences"] == 1:
                longest = case["longest"] = longest * 2 // 3
                case["shortest"] = min(case["shortest"], longest)
        return case
    if op == "attention_cached":
        longest = _log(rng, 1, 65536)
        case = {"op": op, "dtype": dtype, "sequences": _log(rng, 1, 256), "shortest": rng.choice([0, 1, longest]),
                "longest": longest, "heads": heads, "kv_heads": kv, "d": 8 * rng.randint(1, 16),
                "page": rng.choice([16, 32, 64, 128])}
        while case["sequences"] * kv * case["longest"] * case["d"] > 1.2e8:
            case["sequences"] = max(1, case["sequences"] // 2)
            if case["sequences"] == 1:
                case["longest"] = case["longest"] * 2 // 3
                case["shortest"] = min(case["shortest"], case["longest"])
        return case
    if op == "cache_append":
        longest = _log(rng, 1, 2000)
        case = {"op": op, "dtype": dtype, "sequences": _log(rng, 1, 256), "shortest": rng.choice([0, 1, longest]),
                "longest": longest, "held": rng.choice([0, rng.randint(1, 40), rng.randint(1, 2000)]), "kv_heads": kv,
                "d": 8 * rng.randint(1, 16), "page": rng.choice([16, 32, 64, 128])}
        while case["sequences"] > 1 and case["sequences"] * kv * (longest + case["held"]) * case["d"] > 1e7:
            case["sequences"] //= 2
        return case
    rows = _log(rng, 1, 2048)
    vocab = _log(rng, 100, 150000)
    while rows * vocab > 3e7:
        rows = max(1, rows // 2)
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "history": rng.choice([0, _log(rng, 1, 4000)]),
            "states": rng.choice([0, 1, rng.randint(2, 40)]), "bias": rng.random() < 0.5,
            "penalties": rng.random() < 0.7}


def _lengths(case):
    """Each sequence's new tokens and the tokens it held before: plain numbers from the case alone."""
    r = random.Random("%s %d %d %d" % (case["op"], case["sequences"], case["shortest"], case["longest"]))
    n = [r.randint(case["shortest"], case["longest"]) for _ in range(case["sequences"])]
    n[0] = case["longest"]
    if case["op"] == "cache_append":
        return n, [r.randint(case["held"] // 2, case["held"]) for _ in n]
    if case["op"] == "attention_packed":
        more = {"same": lambda x: x, "more": lambda x: x + r.randint(0, 2 * case["longest"]),
                "fewer": lambda x: r.randint(0, x)}[case["keys"]]
        return n, [more(x) for x in n]
    return n, [0] * len(n)


def _history(case):
    r = random.Random("history %d %d" % (case["rows"], case["history"]))
    return [r.randint(0, case["history"]) for _ in range(case["rows"])]


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "attention_packed":
        nq, nk = _lengths(case)
        pairs = 0
        for a, b in zip(nq, nk):
            if not case["causal"]:
                pairs += a * b
            elif b >= a:  # query i sees b - a + 1 + i keys
                pairs += a * (b - a) + a * (a + 1) // 2
            else:
                pairs += b * (b + 1) // 2
        bytes_ = e * case["d"] * (2 * case["heads"] * sum(nq) + 2 * case["kv_heads"] * sum(nk))
        return {"bytes": max(bytes_, 1), "flops": 4 * case["heads"] * case["d"] * pairs}
    if case["op"] == "attention_cached":
        n, _ = _lengths(case)
        blocks = sum(-(-x // case["page"]) for x in n)
        cache = 2 * case["kv_heads"] * (sum(n) * case["d"] + 4 * blocks)
        return {"bytes": cache + 2 * e * case["heads"] * case["d"] * len(n) + 4 * blocks,
                "flops": 4 * case["heads"] * case["d"] * sum(n)}
    if case["op"] == "cache_append":
        n, held = _lengths(case)
        per = 2 * case["kv_heads"] * case["d"]
        # New values read and written in 8 bits; then the touched blocks' values read in 8 bits and written.
        back = sum(a + h % case["page"] for a, h in zip(n, held) if a)
        return {"bytes": max(1, per * (sum(n) * (e + 1) + back * (1 + e))), "flops": per * (3 * sum(n) + back)}
    cells = case["rows"] * case["vocab"]
    words = -(-case["vocab"] // 32)
    bytes_ = 2 * e * cells + 4 * words * min(case["states"], case["rows"]) + 4 * sum(_history(case))
    return {"bytes": bytes_ + (4 * case["vocab"] if case["bias"] else 0), "flops": 4 * cells}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _offsets(n):
    return torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": case}
    if case["op"] == "logit_rules":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (normal(rows, vocab) * 3).to(dt)
        if case["penalties"]:
            n = _history(case)
            s["history_offsets"] = _offsets(n)
            # What was written so far repeats itself: ids crowd towards the low end.
            u = torch.rand(sum(n), device="cuda", generator=g)
            s["history"] = (u.pow(4) * vocab).to(torch.int32).clamp_(max=vocab - 1)
            s["repetition"] = 1 + torch.rand(rows, device="cuda", generator=g)
            s["presence"] = torch.rand(rows, device="cuda", generator=g)
            s["frequency"] = torch.rand(rows, device="cuda", generator=g) / 4
        if case["bias"]:
            s["bias"] = normal(vocab)
        if case["states"]:
            # Grammar states from a few allowed ids to nearly all; some rows are free (-1).
            words = -(-vocab // 32)
            keep = torch.linspace(0.02, 0.95, case["states"], device="cuda")[:, None]
            bits = torch.rand(case["states"], words * 32, device="cuda", generator=g) < keep
            weights = (2 ** torch.arange(32, device="cuda", dtype=torch.int64))
            packed = (bits.view(case["states"], words, 32) * weights).sum(-1)
            s["mask"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
            lo = 0 if case["states"] == 1 else -1
            s["mask_index"] = torch.randint(lo, case["states"], (rows,), device="cuda", generator=g, dtype=torch.int32)
        return s

    n, other = _lengths(case)
    kv, d = case["kv_heads"], case["d"]
    if case["op"] == "attention_packed":
        s["q"] = normal(sum(n), case["heads"], d).to(dt)
        # Keys carry a common direction, as trained projections do, so that the scores are not all alike.
        s["k"] = (normal(sum(other), kv, d) + normal(kv, d)).to(dt)
        s["v"] = normal(sum(other), kv, d).to(dt)
        s["q_offsets"], s["k_offsets"] = _offsets(n), _offsets(other)
        s["longest_q"], s["longest_k"] = max(n), max(other)
        return s

    page = case["page"]
    held = n if case["op"] == "attention_cached" else [a + b for a, b in zip(n, other)]
    blocks = [-(-x // page) for x in held]
    pages = max(1, sum(blocks)) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(n), max(1, max(blocks))), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at: at + b]
        at += b
    s["table"] = table
    for name in ("k", "v"):
        s[name + "_pages"] = torch.randint(-127, 128, (pages, kv, page, d), device="cuda", generator=g).to(torch.int8)
        s[name + "_scales"] = (0.5 + torch.rand(pages, kv, device="cuda", generator=g)) * (3.0 / 127)
    if case["op"] == "attention_cached":
        s["q"] = normal(len(n), case["heads"], d).to(dt)
        s["lengths"] = torch.tensor(n, device="cuda", dtype=torch.int32)
        return s
    s["k_new"] = (normal(sum(n), kv, d) * 1.2).to(dt)
    s["v_new"] = normal(sum(n), kv, d).to(dt)
    s["offsets"] = _offsets(n)
    s["held"] = torch.tensor(other, device="cuda", dtype=torch.int32)
    # Read back from the start of the first block that the new tokens touch.
    first = [h - h % page for h in other]
    s["first"] = torch.tensor(first, device="cuda", dtype=torch.int32)
    s["back_offsets"] = _offsets([h + a - f if a else 0 for a, h, f in zip(n, other, first)])
    s["back"] = sum(h + a - f if a else 0 for a, h, f in zip(n, other, first))
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _packed_rows(offsets, total):
    """For each packed row its sequence and its place in it."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(offsets[1:].long(), row, right=True)
    return seq, row - offsets.long()[seq]


def _softmax_times(scores, allowed, values):
    """sum_j softmax(scores)_j values_j over the allowed j; zero where there is none."""
    scores = scores.masked_fill(~allowed, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == float("-inf"), 0.0)).exp()
    return (p @ values) / p.sum(-1, keepdim=True).clamp_min(torch.finfo(p.dtype).tiny)


def _plain_packed(s):
    c = s["case"]
    kv, d, b = c["kv_heads"], c["d"], c["sequences"]
    group = c["heads"] // kv
    lq, lk = max(1, s["longest_q"]), max(1, s["longest_k"])
    qs, qi = _packed_rows(s["q_offsets"], s["q"].shape[0])
    ks, ki = _packed_rows(s["k_offsets"], s["k"].shape[0])
    q = torch.zeros(b, lq, c["heads"], d, device="cuda")
    k = torch.zeros(b, lk, kv, d, device="cuda")
    v = torch.zeros(b, lk, kv, d, device="cuda")
    q[qs, qi] = s["q"].float()
    k[ks, ki] = s["k"].float()
    v[ks, ki] = s["v"].float()
    q = q.view(b, lq, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, group * lq, d)
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    scores = ((q @ k.transpose(-1, -2)) * d ** -0.5).view(b, kv, group, lq, lk)
    nq, nk = s["q_offsets"].diff(), s["k_offsets"].diff()
    i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    allowed = (j < nk[:, None]).view(b, 1, 1, 1, lk)
    if c["causal"]:
        allowed = allowed & (j <= (i[:, None] + (nk - nq)[:, None, None])).view(b, 1, 1, lq, lk)
    out = _softmax_times(scores.view(b, kv, group, lq, lk), allowed, v.unsqueeze(2))
    return out.permute(0, 3, 1, 2, 4).reshape(b, lq, c["heads"], d)[qs, qi].to(s["q"].dtype)


def _plain_cached(s):
    c = s["case"]
    kv, d, b, page = c["kv_heads"], c["d"], c["sequences"], c["page"]
    table = s["table"].clamp_min(0).long()
    k = (s["k_pages"][table].float() * s["k_scales"][table][..., None, None]).transpose(1, 2).reshape(b, kv, -1, d)
    v = (s["v_pages"][table].float() * s["v_scales"][table][..., None, None]).transpose(1, 2).reshape(b, kv, -1, d)
    q = s["q"].float().view(b, kv, -1, d)
    scores = (q @ k.transpose(-1, -2)) * d ** -0.5
    j = torch.arange(table.shape[1] * page, device="cuda")
    out = _softmax_times(scores, (j < s["lengths"][:, None]).view(b, 1, 1, -1), v)
    return out.reshape(b, c["heads"], d).to(s["q"].dtype)


def _plain_append(s, name):
    """The new tokens join their blocks: a block's scale is the largest magnitude it has seen / 127, and what it
    held before is rounded again where the scale grows.  Decisions next to a rounding border are taken in 64 bits."""
    page = s["case"]["page"]
    new, pages, scales = s[name + "_new"], s[name + "_pages"], s[name + "_scales"]
    seq, i = _packed_rows(s["offsets"], new.shape[0])
    held = s["held"].long()
    at = held[seq] + i
    where = s["table"].long()[seq, at // page]
    x = new.float()
    amax = torch.zeros_like(scales)
    amax.scatter_reduce_(0, where[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    part = torch.nonzero((held % page > 0) & (s["offsets"].diff() > 0)).squeeze(1)  # sequences with a part-filled block
    old_page = s["table"].long()[part, held[part] // page]
    before = torch.zeros_like(scales)
    before[old_page] = scales[old_page]
    grown = torch.maximum(before, amax * (1.0 / 127))
    touched = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda")
    touched[where] = True
    scales.copy_(torch.where(touched[:, None], grown, scales))
    ratio = before[old_page].double(), scales[old_page].double()
    again = (pages[old_page].double() * ratio[0][..., None, None] / ratio[1][..., None, None]).round().to(torch.int8)
    mine = (torch.arange(page, device="cuda") < (held[part] % page)[:, None])[:, None, :, None]
    move = mine & (ratio[1] > ratio[0])[..., None, None]
    pages[old_page] = torch.where(move, again, pages[old_page])
    sc = scales[where].double()[..., None]
    pages[where, :, at % page] = torch.where(sc > 0, x.double() / sc, 0.0).round().clamp(-127, 127).to(torch.int8)


def _plain_read(s, name):
    page = s["case"]["page"]
    seq, i = _packed_rows(s["back_offsets"], s["back"])
    at = s["first"].long()[seq] + i
    where = s["table"].long()[seq, at // page]
    return (s[name + "_pages"][where, :, at % page].float() * s[name + "_scales"][where][..., None]).to(s["k_new"].dtype)


def _plain_rules(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    if "history" in s:
        seq, _ = _packed_rows(s["history_offsets"], s["history"].numel())
        counts = torch.zeros(rows * vocab, device="cuda")
        counts.scatter_add_(0, seq * vocab + s["history"].long(), torch.ones_like(seq, dtype=torch.float32))
        counts = counts.view(rows, vocab)
        seen = counts > 0
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * counts - s["presence"][:, None] * seen
    if "bias" in s:
        x = x + s["bias"]
    if "mask" in s:
        ids = torch.arange(vocab, device="cuda")
        state = s["mask_index"].long()
        words = s["mask"][state.clamp_min(0)][:, ids // 32]
        allowed = ((words >> (ids % 32)) & 1).bool() | (state < 0)[:, None]
        x = x.masked_fill(~allowed, float("-inf"))
    return x.to(s["logits"].dtype)


def run(s):
    op = s["case"]["op"]
    if not own:
        if op == "attention_packed":
            return _plain_packed(s)
        if op == "attention_cached":
            return _plain_cached(s)
        if op == "logit_rules":
            return _plain_rules(s)
        _plain_append(s, "k")
        _plain_append(s, "v")
        return [_plain_read(s, "k"), _plain_read(s, "v"), s["k_scales"], s["v_scales"]]
    P, gpu = _gpu()
    stream = torch.cuda.current_stream()
    if op == "attention_packed":
        return gpu.attention_packed(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], torch.empty_like(s["q"]),
                                    causal=s["case"]["causal"], stream=stream)
    if op == "logit_rules":
        return gpu.logit_rules(s["logits"], torch.empty_like(s["logits"]), history=s.get("history"),
                               history_offsets=s.get("history_offsets"), repetition=s.get("repetition"),
                               presence=s.get("presence"), frequency=s.get("frequency"), bias=s.get("bias"),
                               mask=s.get("mask"), mask_index=s.get("mask_index"), stream=stream)
    cache = P.PagedCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    if op == "attention_cached":
        return gpu.attention_cached(cache, s["q"], s["lengths"], s["table"], torch.empty_like(s["q"]), stream=stream)
    gpu.cache_append(cache, s["k_new"], s["v_new"], s["offsets"], s["held"], s["table"], stream=stream)
    k = torch.empty(s["back"], *s["k_new"].shape[1:], dtype=s["k_new"].dtype, device="cuda")
    v = torch.empty_like(k)
    gpu.cache_read(cache, k, v, s["back_offsets"], s["first"], s["table"], stream=stream)
    return [k, v, s["k_scales"], s["v_scales"]]


# ---------------------------------------------------------------------------
# The definitions in 64 bits, one sequence, block or row at a time
# ---------------------------------------------------------------------------

def _attend(q, k, v, first):
    """q [n, heads, d], k / v [m, kv, d] in float64; query i sees keys 0 .. first + i (all with first None)."""
    n, heads, d = q.shape
    m, kv = k.shape[:2]
    out = torch.zeros_like(q)
    if n == 0 or m == 0:
        return out
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        for a in range(0, n, 4096):
            z = torch.einsum("id,jd->ij", q[a:a + 4096, h], kh) / math.sqrt(d)
            if first is not None:
                last = torch.arange(a, a + z.shape[0], device="cuda")[:, None] + first
                z[torch.arange(m, device="cuda")[None] > last] = -math.inf
            w = torch.softmax(z, -1).nan_to_num(0.0)
            out[a:a + 4096, h] = w @ vh
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention_packed":
        nq, nk = _lengths(case)
        parts, a, b = [], 0, 0
        for x, y in zip(nq, nk):
            parts.append(_attend(s["q"][a:a + x].double(), s["k"][b:b + y].double(), s["v"][b:b + y].double(),
                                 y - x if case["causal"] else None))
            a, b = a + x, b + y
        return torch.cat(parts)
    if case["op"] == "attention_cached":
        parts = []
        for i, x in enumerate(_lengths(case)[0]):
            rows = s["table"][i, : -(-x // case["page"])].long()
            k, v = ((s[m + "_pages"][rows].double() * s[m + "_scales"][rows].double()[..., None, None])
                    .permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["d"])[:x] for m in ("k", "v"))
            parts.append(_attend(s["q"][i:i + 1].double(), k, v, None))
        return torch.cat(parts)
    if case["op"] == "cache_append":
        return _exact_append(case, s)
    x = s["logits"].double()
    if "history" in s:
        edge = s["history_offsets"].tolist()
        for r in range(case["rows"]):
            ids, times = torch.unique(s["history"][edge[r]:edge[r + 1]].long(), return_counts=True)
            y, rep = x[r, ids], s["repetition"][r].double()
            y = torch.where(y > 0, y / rep, y * rep)
            x[r, ids] = y - times * s["frequency"][r].double() - s["presence"][r].double()
    if "bias" in s:
        x += s["bias"].double()
    if "mask" in s:
        shift = torch.arange(32, device="cuda", dtype=torch.int32)
        bits = ((s["mask"][:, :, None] >> shift) & 1).flatten(1)[:, : case["vocab"]] == 0
        for r, state in enumerate(s["mask_index"].tolist()):
            if state >= 0:
                x[r, bits[state]] = -math.inf
    return x


def _exact_append(case, s):
    n, held = _lengths(case)
    page, outs, scales = case["page"], [], []
    table = s["table"].tolist()
    for m in ("k", "v"):
        x, sc, values, at = s[m + "_new"].double(), s[m + "_scales"].clone(), [], 0
        for i, (a, h) in enumerate(zip(n, held)):
            pos = h
            while pos < h + a:
                blk, lo = table[i][pos // page], pos % page
                hi = min(page, lo + h + a - pos)
                new = x[at:at + hi - lo]
                before = sc[blk].clone() if lo else torch.zeros_like(sc[blk])
                # A scale is a 32-bit number by definition; what is divided by it is not rounded first.
                now = torch.maximum(before, new.abs().amax((0, 2)).float() * torch.tensor(1 / 127).cuda())
                old = s[m + "_pages"][blk].double()[:, :lo]
                old = torch.where((now > before)[:, None, None],
                                  (old * before.double()[:, None, None] / now.double()[:, None, None]).round(), old)
                fresh = (new.transpose(0, 1) / now.double()[:, None, None]).nan_to_num(0.0).round()
                values.append((torch.cat([old, fresh], 1) * now.double()[:, None, None]).transpose(0, 1))
                sc[blk] = now
                pos, at = pos + hi - lo, at + hi - lo
        outs.append(torch.cat(values) if values else x[:0])
        scales.append(sc.double())
    return outs + scales
