"""Single operators as cases to time and to compare: a paged key/value cache held in 8 bits, the attention that reads it, and
the log-probabilities of given tokens.

A case names its operator (`op`):

  append     the keys and values of a step's new tokens, quantised into their pages
  read       cached keys and values of some requests, back as dense rows
  decode     attention of single tokens over the cache
  prompt     attention of prompt portions over the cache, their own keys appended before
  logprobs   log-probability of one given token a row, the row's entropy and its likeliest tokens

The cache is [num_pages, key/value heads, page size, head size] codes of `code` ("float8_e4m3fn" or "int8") for keys and for
values, with one float32 scale for each page and head; a scale is the smallest power of two by which the largest value of
its block fits the code, so that a block that grows is brought to its new scale by a power of two.

`run` computes an operator in its plain form with elementary torch operations in 32 bits, or, where the module's `own` is
true, calls the framework's kernels.  Sizes are those of configs/*.json, of the test models and of requests that a server
has in flight at a time; beside them generic layouts of grouped heads.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
CODES = {"float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
SMALLEST_EXPONENT = -100         # of a scale: what a block of zeros has


def _kv(name, op, code, dtype, requests, heads, kv_heads, head_dim, page, before, new, **more):
    """before, new: (shortest, longest) numbers of tokens a request has in the cache, and brings."""
    return dict(name=name, op=op, code=code, dtype=dtype, requests=requests, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                before_lo=before[0], before_hi=before[1], new_lo=new[0], new_hi=new[1],
                **dict(dict(window=0, keep_first=0, softcap=0.0, sink=False), **more))


def _rows(name, dtype, rows, vocab, top):
    return dict(name=name, op="logprobs", dtype=dtype, rows=rows, vocab=vocab, top=top)


def listed():
    return [
        # a decode step of a few GPT-2 small requests: one layer's new keys and values, where latency counts
        _kv("append_step_8", "append", "float8_e4m3fn", "bfloat16", 8, 12, 12, 64, 16, (100, 900), (1, 1)),
        # ragged prompts admitted together, GPT-2 xl: bytes count
        _kv("append_prompts_xl_int8", "append", "int8", "bfloat16", 24, 25, 25, 64, 16, (0, 90), (400, 930)),
        # one request's cache back in 32 bits, as a check or a kernel without an 8-bit form wants it
        _kv("read_one_fp32", "read", "int8", "float32", 1, 12, 12, 64, 16, (700, 700), (0, 0)),
        # the caches of many requests back in bfloat16, grouped heads
        _kv("read_many", "read", "float8_e4m3fn", "bfloat16", 24, 32, 8, 128, 16, (300, 4000), (0, 0)),
        # a decode step of a few GPT-2 small requests
        _kv("decode_8", "decode", "float8_e4m3fn", "bfloat16", 8, 12, 12, 64, 16, (100, 900), (1, 1)),
        # a server's decode step of GPT-2 xl with many requests of different ages
        _kv("decode_64_xl_int8", "decode", "int8", "bfloat16", 64, 25, 25, 64, 16, (64, 1000), (1, 1)),
        # a few requests with very long contexts, grouped heads: the cache's bytes are the time
        _kv("decode_long", "decode", "float8_e4m3fn", "bfloat16", 4, 32, 8, 128, 16, (30000, 100000), (1, 1)),
        # the 32-bit path with a window, kept first tokens and a sink, heads of an odd size, small pages
        _kv("decode_window_fp32", "decode", "int8", "float32", 24, 16, 4, 80, 8, (500, 6000), (1, 1), window=1500, keep_first=4, sink=True),
        # prompts of GPT-2 small that nearly fill its context
        _kv("prompts_4", "prompt", "float8_e4m3fn", "bfloat16", 4, 12, 12, 64, 16, (0, 60), (500, 950)),
        # a portion of a long prompt behind what came before it, grouped heads
        _kv("prompt_portion_long", "prompt", "int8", "bfloat16", 1, 32, 8, 128, 16, (6000, 6000), (2048, 2048)),
        # what a decode step returns beside its tokens
        _rows("logprobs_step_8", "float32", 8, 50257, 5),
        # a scored text: every token of two prompts that fill the context
        _rows("logprobs_text", "float32", 2046, 50257, 20),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([50257, 50304, 32000, 1000, 512, 128256, _log_int(rng, 300, 150000)])
        rows = max(1, min(_log_int(rng, 1, 4000), 2046 * 50257 // vocab))
        c = _rows("", rng.choice(["float32", "float32", "bfloat16"]), rows, vocab, rng.choice([1, 5, 20, rng.randint(1, 32)]))
    else:
        code, dtype = rng.choice(list(CODES)), rng.choice(["bfloat16", "bfloat16", "float32"])
        kv_heads = rng.choice([1, 2, 4, 8, 12, 25, rng.randint(1, 16)])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8, rng.randint(1, 12)])
        head_dim, page = rng.choice([64, 64, 128, 128, 16, 48, 80, 96, 256]), rng.choice([16, 16, 16, 8, 32, 64])
        requests = _log_int(rng, 1, 64)
        more = {}
        if op in ("decode", "prompt"):
            if rng.random() < 0.3:
                more = dict(window=_log_int(rng, 8, 2000), keep_first=rng.choice([0, 0, 4, 20]), sink=rng.random() < 0.5)
            elif rng.random() < 0.15:
                more = dict(softcap=rng.choice([20.0, 50.0]))
        width = kv_heads * head_dim
        if op == "decode":
            most = min(100000, 64 * 1000 * 1600 // (requests * width))       # keys a request may have
            hi = max(2, _log_int(rng, 2, max(3, most)))
            before, new = (max(1, hi // rng.randint(1, 8)), hi), (1, 1)
        elif op == "prompt":
            requests = min(requests, 12)
            # no more products, and no more scores, than the longest listed portion has
            most = int(math.sqrt(min(2.0e11 / head_dim, 2.6e8) / (requests * heads)))
            hi = max(2, _log_int(rng, 2, max(3, min(4000, most))))
            new = (max(1, hi // rng.randint(1, 6)), hi)
            hi = rng.choice([0, _log_int(rng, 1, max(2, min(6000, most)))])
            before = (hi // 2, hi)
        else:
            most = max(2, min(4000, 24 * 4000 * 1024 // (2 * requests * width)))
            hi = max(1, _log_int(rng, 1, most))
            pair = (max(1, hi // rng.randint(1, 6)), hi)
            before, new = (pair, (0, 0)) if op == "read" else (rng.choice([(0, 0), (0, 90), (1, 500)]), pair if rng.random() < 0.6 else (1, 1))
        c = _kv("", op, code, dtype, requests, heads, kv_heads, head_dim, page, before, new, **more)
    del c["name"]
    return c


def _lengths(case):
    """(tokens a request has, tokens it brings): the same for every seed, so that a case has one amount of work."""
    r = np.random.RandomState(case["requests"] * 7919 + case["before_hi"] * 31 + case["new_hi"])
    before = r.randint(case["before_lo"], case["before_hi"] + 1, case["requests"])
    new = r.randint(case["new_lo"], case["new_hi"] + 1, case["requests"])
    before[0], new[0] = case["before_hi"], case["new_hi"]
    return before.tolist(), new.tolist()


def _seen(case, before, new):
    """Keys that each new token sees, as a list over the tokens."""
    seen = []
    for b, n in zip(before, new):
        pos = np.arange(b, b + n)
        lo = np.maximum(0, pos + 1 - case["window"]) if case["window"] else np.zeros_like(pos)
        seen.append(pos + 1 - lo + np.minimum(case["keep_first"], lo))
    return np.concatenate(seen)


def work(case):
    if case["op"] == "logprobs":
        es = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * es + 4 * 3 + 8 * case["top"]), "flops": case["rows"] * case["vocab"] * 5}
    before, new = _lengths(case)
    es, kv, page = (4 if case["dtype"] == "float32" else 2), case["kv_heads"] * case["head_dim"], case["page"]
    blocks = lambda tokens: -(-tokens // page)        # noqa: E731
    if case["op"] == "append":
        n = sum(new)
        touched = sum(blocks(b + m) - b // page for b, m in zip(before, new))
        return {"bytes": 2 * (n * kv * (es + 1) + touched * case["kv_heads"] * 4), "flops": 2 * n * kv * 3}
    if case["op"] == "read":
        n = sum(before)
        return {"bytes": 2 * (n * kv * (es + 1) + sum(blocks(b) for b in before) * case["kv_heads"] * 4), "flops": 2 * n * kv}
    n = sum(new)
    # a key that any of a request's new tokens sees is read once, with its value
    keys = sum(int(min(b + m, (case["window"] + m - 1 + case["keep_first"]) if case["window"] else b + m)) for b, m in zip(before, new))
    return {"bytes": 2 * keys * kv + 2 * blocks(keys) * case["kv_heads"] * 4 + 2 * n * case["heads"] * case["head_dim"] * es,
            "flops": 4 * int(_seen(case, before, new).sum()) * case["heads"] * case["head_dim"]}


# ---- the quantisation ------------------------------------------------------------------------------------------
def _scale_of(amax, code):
    """The smallest power of two s with amax <= largest * s, from amax = m * 2^e with m in [0.5, 1)."""
    m, e = torch.frexp(amax)
    top_m, top_e = math.frexp(LARGEST[code])
    e = torch.where(amax > 0, e - top_e + (m > top_m).to(e.dtype), SMALLEST_EXPONENT).clamp(min=SMALLEST_EXPONENT)
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _code(x, code):
    return torch.round(x).to(torch.int8) if code == torch.int8 else x.to(code)


def _take(codes, index):
    """codes[index] for types that torch does not index, as float32."""
    return codes.view(torch.uint8)[index].view(codes.dtype).float()


def _put(codes, index, values):
    codes.view(torch.uint8)[index] = values.view(torch.uint8)


# ---- inputs ------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)        # noqa: E731
    dtype = TYPES[case["dtype"]]
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], min(case["top"], case["vocab"])
        logits = (randn(n, v) * (1.0 + 2.0 * torch.rand(n, 1, generator=g, device=DEV)) - 30.0).to(dtype)
        # half of the given tokens are likely ones, as those of a text are
        likely = logits.argmax(dim=1)
        given = torch.where(torch.rand(n, generator=g, device=DEV) < 0.5, likely, torch.randint(0, v, (n,), generator=g, device=DEV))
        empty = lambda *shape, t=torch.float32: torch.empty(*shape, dtype=t, device=DEV)        # noqa: E731
        return dict(op="logprobs", logits=logits, ids=given.to(torch.int32), top=k, logprob=empty(n), entropy=empty(n),
                    top_ids=empty(n, k, t=torch.int32), top_logprobs=empty(n, k))
    code, op = CODES[case["code"]], case["op"]
    H, Hkv, D, ps, S = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["requests"]
    before, new = _lengths(case)
    blocks = [max(1, -(-(b + n) // ps)) for b, n in zip(before, new)]
    P = sum(blocks) + 3
    # pages in the order of a pool that requests of different ages have used; a prompt's tend to be a run
    order = torch.randperm(P, generator=g, device=DEV) if op != "prompt" else torch.arange(P, device=DEV)
    start = np.cumsum([0] + blocks[:-1])
    at = torch.tensor(start, device=DEV)[:, None] + torch.arange(max(blocks), device=DEV)[None, :]
    has = torch.arange(max(blocks), device=DEV)[None, :] < torch.tensor(blocks, device=DEV)[:, None]
    table = torch.where(has, order[at.clamp(max=P - 1)], -1).to(torch.int32).contiguous()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)        # noqa: E731
    s = dict(op=op, code=code, dtype=dtype, H=H, Hkv=Hkv, D=D, ps=ps, table=table, before=i32(before), new=i32(new),
             q_start=i32(np.cumsum([0] + new).tolist()), max_new=max(new), max_before=max(before), rule={}, sink=None)
    # cached keys and values: some channels are larger than others, and blocks differ in size
    for which in ("k", "v"):
        channel = torch.exp(0.5 * randn(1, Hkv, 1, D))
        codes = torch.empty(P, Hkv, ps, D, dtype=code, device=DEV)
        scales = torch.empty(P, Hkv, device=DEV)
        step = max(1, (1 << 26) // (Hkv * ps * D))
        for p in range(0, P, step):
            x = randn(min(step, P - p), Hkv, ps, D) * channel * torch.exp(0.3 * randn(min(step, P - p), Hkv, 1, 1))
            sc = _scale_of(x.abs().amax(dim=(2, 3)), code)
            codes[p:p + step] = _code(x / sc[..., None, None], code)
            scales[p:p + step] = sc
        s[which], s[which + "_scale"] = codes, scales
    if op == "append":
        # the new keys and values are columns of one fused product, as the engine has them
        qkv = (randn(sum(new), (H + 2 * Hkv) * D) * torch.exp(0.5 * randn(1, (H + 2 * Hkv) * D))).to(dtype)
        s["k_src"], s["v_src"] = qkv[:, H * D:(H + Hkv) * D], qkv[:, (H + Hkv) * D:]
    elif op == "read":
        n = sum(before)
        s["out_start"] = i32(np.cumsum([0] + before).tolist())
        s["first"] = i32([0] * S)
        s["k_out"], s["v_out"] = (torch.empty(n, Hkv * D, dtype=dtype, device=DEV) for _ in range(2))
    else:
        n = sum(new)
        s["q"] = (randn(n, H * D) * 1.5).to(dtype)
        s["out"] = torch.empty(n, H * D, dtype=dtype, device=DEV)
        s["scale"] = 1.0 / math.sqrt(D)
        s["rule"] = dict(window=case["window"], keep_first=case["keep_first"], softcap=case["softcap"])
        s["sink"] = randn(H) if case["sink"] else None
        s["token_seq"] = torch.arange(S, dtype=torch.int32, device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return (_own if own else _plain)[state["op"]](state)


def _plain_append(s):
    seq = torch.repeat_interleave(torch.arange(s["before"].numel(), device=DEV), s["new"].long(), output_size=s["k_src"].shape[0])
    pos = s["before"][seq] + torch.arange(seq.numel(), device=DEV) - s["q_start"][seq]
    page, slot = s["table"][seq, pos // s["ps"]].long(), pos % s["ps"]
    # pages that hold earlier tokens of their request: their blocks grow
    old, kept = s["table"][torch.arange(s["before"].numel(), device=DEV), s["before"] // s["ps"]].long(), s["before"] % s["ps"]
    holds = torch.zeros(s["k"].shape[0], 1, dtype=torch.bool, device=DEV)
    holds[old, 0] = kept > 0
    touched = torch.zeros_like(holds)
    touched[page] = True
    for_old = torch.arange(s["ps"], device=DEV)[None, None, :, None] < kept[:, None, None, None]
    return {"k": _plain_append_one(s, "k", page, slot, old, holds, touched, for_old), "k_scale": s["k_scale"],
            "v": _plain_append_one(s, "v", page, slot, old, holds, touched, for_old), "v_scale": s["v_scale"]}


def _plain_append_one(s, which, page, slot, old, holds, touched, for_old):
    codes, scales, code = s[which], s[which + "_scale"], s["code"]
    x = s[which + "_src"].float().reshape(-1, s["Hkv"], s["D"])
    amax = torch.zeros_like(scales).index_reduce_(0, page, x.abs().amax(dim=2), "amax")
    need = _scale_of(amax, code)
    now = torch.where(holds, torch.maximum(need, scales), need)
    had = codes.view(torch.uint8)[old]
    again = _code(had.view(code).float() * (scales / now)[old][..., None, None], code).view(torch.uint8)
    _put(codes, old, torch.where(for_old, again, had))
    _put(codes, (page, slice(None), slot), _code(x / now[page][..., None], code))
    scales.copy_(torch.where(touched, now, scales))
    return codes


def _plain_read(s):
    seq = torch.repeat_interleave(torch.arange(s["before"].numel(), device=DEV), s["before"].long(), output_size=s["k_out"].shape[0])
    pos = s["first"][seq] + torch.arange(seq.numel(), device=DEV) - s["out_start"][seq]
    page, slot = s["table"][seq, pos // s["ps"]].long(), pos % s["ps"]
    k = _take(s["k"], (page, slice(None), slot)) * s["k_scale"][page][..., None]
    v = _take(s["v"], (page, slice(None), slot)) * s["v_scale"][page][..., None]
    return {"k": k.flatten(1).to(s["dtype"]), "v": v.flatten(1).to(s["dtype"])}


def _plain_attention(s):
    """Every request's keys side by side, its new tokens padded to the most that one brings."""
    S, H, Hkv, D, n = s["before"].numel(), s["H"], s["Hkv"], s["D"], s["max_new"]
    pages = s["table"].long().clamp(min=0)
    k, v = ((_take(s[w], pages) * s[w + "_scale"][pages][..., None, None]).permute(0, 2, 1, 3, 4).reshape(S, Hkv, -1, D) for w in ("k", "v"))
    row = s["q_start"][:-1, None] + torch.arange(n, device=DEV)[None, :]
    mine = torch.arange(n, device=DEV)[None, :] < s["new"][:, None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].float().reshape(S, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).reshape(S, H, n, -1)
    if s["rule"]["softcap"]:
        score = s["rule"]["softcap"] * torch.tanh(score / s["rule"]["softcap"])
    j = torch.arange(score.shape[-1], device=DEV)[None, None, :]
    pos = (s["before"][:, None] + torch.arange(n, device=DEV)[None, :])[..., None]
    sees = j <= pos
    if s["rule"]["window"]:
        sees &= (j > pos - s["rule"]["window"]) | (j < s["rule"]["keep_first"])
    score = score.masked_fill_(~sees[:, None], float("-inf"))
    most = score.amax(dim=-1, keepdim=True)
    p = score.sub_(most).exp_()
    total = p.sum(dim=-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"][None, :, None, None] - most)
    out = torch.matmul(p.reshape(S, Hkv, -1, p.shape[-1]), v).reshape(S, H, n, D) / total
    return out.permute(0, 2, 1, 3)[mine].reshape(-1, H * D).to(s["dtype"])


def _plain_logprobs(s):
    x = s["logits"].float()
    best = x.amax(dim=1, keepdim=True)
    d = x - best
    e = torch.exp(d)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    value, index = torch.sort(d, dim=1, descending=True, stable=True)
    return {"logprob": d.gather(1, s["ids"].long()[:, None])[:, 0] - log_total, "entropy": log_total - (e * d).sum(dim=1) / total,
            "top_ids": index[:, :s["top"]].to(torch.int32), "top_logprobs": value[:, :s["top"]] - log_total[:, None]}


def _cache(s):
    from sandyrt_b200.csrc import ops

    return ops.Cache8(s["k"], s["v"], s["k_scale"], s["v_scale"])


def _own_append(s):
    from sandyrt_b200.csrc import ops

    ops.kv_append_8bit(s["k_src"], s["v_src"], _cache(s), s["table"], s["q_start"], s["before"], max_q_len=s["max_new"])
    return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"]}


def _own_read(s):
    from sandyrt_b200.csrc import ops

    ops.kv_read_8bit(_cache(s), s["table"], s["first"], s["out_start"], s["k_out"], s["v_out"], max_len=s["max_before"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_decode(s):
    from sandyrt_b200.csrc import ops

    ops.decode_attention_8bit(s["q"], _cache(s), s["table"], s["token_seq"], s["before"], s["out"], n_heads=s["H"], scale=s["scale"],
                              sink=s["sink"], **s["rule"])
    return s["out"]


def _own_prompt(s):
    from sandyrt_b200.csrc import ops

    ops.prefill_attention_8bit(s["q"], _cache(s), s["table"], s["q_start"], s["before"], s["out"], n_heads=s["H"], max_q_len=s["max_new"],
                               scale=s["scale"], sink=s["sink"], **s["rule"])
    return s["out"]


def _own_logprobs(s):
    from sandyrt_b200.csrc import ops

    ops.token_logprobs(s["logits"], s["ids"], s["logprob"], entropy=s["entropy"], top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
    return {"logprob": s["logprob"], "entropy": s["entropy"], "top_ids": s["top_ids"], "top_logprobs": s["top_logprobs"]}


_plain = dict(append=_plain_append, read=_plain_read, decode=_plain_attention, prompt=_plain_attention, logprobs=_plain_logprobs)
_own = dict(append=_own_append, read=_own_read, decode=_own_decode, prompt=_own_prompt, logprobs=_own_logprobs)


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "decode": _exact_attention, "prompt": _exact_attention,
            "logprobs": _exact_logprobs}[s["op"]](s)


def _nearest(y, code):
    """The code's value nearest to y, ties to the even one: e4m3 has four significant bits down to 2^-6 and steps of 2^-9 below."""
    if code == torch.int8:
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_append(s):
    got = {}
    before, new, table, ps, code = s["before"].tolist(), s["new"].tolist(), s["table"].tolist(), s["ps"], s["code"]
    for w in ("k", "v"):
        codes, scales = s[w].to(torch.float64), s[w + "_scale"].double()
        x = s[w + "_src"].double().reshape(-1, s["Hkv"], s["D"])
        t = 0
        for b, n, pages in zip(before, new, table):
            for first in range(b // ps * ps, b + n, ps):
                lo, hi = max(first, b), min(first + ps, b + n)
                page, kept = pages[first // ps], lo - first
                rows = x[t + lo - b:t + hi - b].transpose(0, 1)                    # [Hkv, tokens, D]
                amax = rows.abs().amax(dim=(1, 2))
                e = torch.ceil(torch.log2((amax / LARGEST[code]).clamp(min=2.0 ** SMALLEST_EXPONENT)))
                e = torch.where(torch.exp2(e) * LARGEST[code] < amax, e + 1, e)
                e = torch.where((torch.exp2(e - 1) * LARGEST[code] >= amax) & (e > SMALLEST_EXPONENT), e - 1, e)
                now = torch.exp2(e)
                if kept:
                    now = torch.maximum(now, scales[page])
                    codes[page, :, :kept] = _nearest(codes[page, :, :kept] * (scales[page] / now)[:, None, None], code)
                codes[page, :, kept:kept + hi - lo] = _nearest(rows / now[:, None, None], code)
                scales[page] = now
            t += n
        got[w], got[w + "_scale"] = codes, scales
    return got


def _exact_read(s):
    got = {}
    for w in ("k", "v"):
        rows = []
        for n, pages in zip(s["before"].tolist(), s["table"]):
            pages = pages[:-(-n // s["ps"])].long()
            x = s[w].view(torch.uint8)[pages].view(s["code"]).double() * s[w + "_scale"].double()[pages][..., None, None]
            rows.append(x.transpose(1, 2).reshape(-1, s["Hkv"] * s["D"])[:n])
        got[w] = torch.cat(rows)
    return got


def _exact_attention(s):
    H, Hkv, D, ps = s["H"], s["Hkv"], s["D"], s["ps"]
    out = []
    for r, (b, n) in enumerate(zip(s["before"].tolist(), s["new"].tolist())):
        pages = s["table"][r, :-(-(b + n) // ps)].long()
        k, v = ((s[w].view(torch.uint8)[pages].view(s["code"]).double() * s[w + "_scale"].double()[pages][..., None, None])
                .transpose(0, 1).reshape(Hkv, -1, D)[:, :b + n] for w in ("k", "v"))
        t = int(s["q_start"][r])
        q = s["q"][t:t + n].double().reshape(n, H, D).transpose(0, 1)
        pos = torch.arange(b, b + n, device=DEV)[:, None]
        j = torch.arange(b + n, device=DEV)[None, :]
        hidden = j > pos
        if s["rule"]["window"]:
            hidden |= (j <= pos - s["rule"]["window"]) & (j >= s["rule"]["keep_first"])
        heads = []
        for h in range(H):
            x = q[h] @ k[h * Hkv // H].T * s["scale"]
            if s["rule"]["softcap"]:
                x = torch.tanh(x / s["rule"]["softcap"]) * s["rule"]["softcap"]
            x[hidden] = float("-inf")
            extra = [] if s["sink"] is None else [s["sink"][h].double().expand(n, 1)]
            lse = torch.logsumexp(torch.cat([x] + extra, dim=1), dim=1, keepdim=True)
            heads.append(torch.exp(x - lse) @ v[h * Hkv // H])
        out.append(torch.stack(heads, dim=1).reshape(n, H * D))
    return torch.cat(out)


def _exact_logprobs(s):
    n, k = s["logits"].shape[0], s["top"]
    got = {"logprob": [], "entropy": [], "top_logprobs": []}
    for r in range(0, n, 256):
        x = s["logits"][r:r + 256].double()
        lp = x - torch.logsumexp(x, dim=1, keepdim=True)
        got["logprob"].append(lp.gather(1, s["ids"][r:r + 256].long()[:, None])[:, 0])
        got["entropy"].append(-(lp.exp() * lp).sum(dim=1))
        got["top_logprobs"].append(lp.topk(k, dim=1).values)
    return {w: torch.cat(v) for w, v in got.items()} | {"top_ids": None}
