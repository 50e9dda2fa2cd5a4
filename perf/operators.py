"""Workloads of the serving operators: prompt attention, the quantised key/value cache (append and
read back), the batched single-token attention that reads it, and token sampling.

``run`` computes a case with elementary torch operations (``own`` false) or through
``qmoe_b200.serving`` (``own`` true).  ``exact`` states the same results in 64 bits, written apart.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ---- cases ---------------------------------------------------------------------------------------
def listed():
    return [
        # the generation benchmark's prompt: one sequence of 128 ids, 32 heads of 65 values
        {"name": "prompt_single_128", "op": "prompt", "seqs": 1, "total": 128, "prefix": 0, "heads": 32,
         "kv_heads": 32, "dim": 65, "dtype": "bf16", "bias": 0, "layout": 1},
        # requests of uneven lengths that arrive together, grouped heads, one of them a single token
        {"name": "prompt_packed_8k", "op": "prompt", "seqs": 16, "total": 8192, "prefix": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "bias": 0, "layout": 2},
        # one long document
        {"name": "prompt_long_16k", "op": "prompt", "seqs": 1, "total": 16384, "prefix": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "bias": 0, "layout": 3},
        # Switch attention: unscaled, relative-position bias, the later part of prompts fed in pieces
        {"name": "prompt_bias_pieces", "op": "prompt", "seqs": 5, "total": 2049, "prefix": 777, "heads": 12,
         "kv_heads": 12, "dim": 64, "dtype": "fp16", "bias": 128, "layout": 4},
        # prompts entering the cache
        {"name": "append_prompts_16k", "op": "append", "seqs": 8, "total": 16384, "past": 0, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "format": "e4m3", "page": 64, "layout": 5},
        # one decoding step of a batch entering the cache
        {"name": "append_step_64", "op": "append", "seqs": 64, "total": 64, "past": 500, "kv_heads": 32,
         "dim": 65, "dtype": "bf16", "format": "int8", "page": 16, "layout": 6},
        # a cache handed to a consumer that wants 16-bit keys and values
        {"name": "read_back_64k", "op": "read", "seqs": 16, "total": 65536, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "format": "e4m3", "page": 64, "layout": 7},
        {"name": "read_back_ragged", "op": "read", "seqs": 9, "total": 1111, "kv_heads": 32, "dim": 65,
         "dtype": "fp16", "format": "int8", "page": 16, "layout": 8},
        # a decoding step of one sequence with the generation benchmark's heads
        {"name": "decode_single_1k", "op": "decode", "seqs": 1, "total": 1000, "heads": 32, "kv_heads": 32,
         "dim": 65, "dtype": "bf16", "format": "int8", "page": 16, "bias": 128, "layout": 9},
        # a decoding step of a large batch with grouped heads
        {"name": "decode_batch_64", "op": "decode", "seqs": 64, "total": 262144, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "format": "e4m3", "page": 64, "bias": 0, "layout": 10},
        # the end of a decoding step: few rows over the generation benchmark's vocabulary
        {"name": "sample_4", "op": "sample", "rows": 4, "vocab": 32128, "dtype": "fp32", "mode": "all", "layout": 11},
        # the same for a large batch over a large vocabulary, every row with its own settings
        {"name": "sample_256", "op": "sample", "rows": 256, "vocab": 131072, "dtype": "fp32", "mode": "mixed",
         "layout": 12},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm, odd ones among them."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "append", "read", "decode", "decode", "sample"])
    layout = rng.randrange(1 << 20)
    kv = rng.choice([1, 2, 3, 8, 12, 32])
    dim = rng.choice([16, 40, 64, 65, 80, 96, 127, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    fmt, page = rng.choice(["e4m3", "int8"]), rng.choice([16, 32, 64, 128])
    if op == "prompt":
        group = rng.choice([1, 2, 3, 4, 8])
        group = max(1, min(group, 32 // kv))
        total = _spread(rng, 1, 12000)
        return {"op": op, "seqs": min(total, _spread(rng, 1, 40)), "total": total, "prefix": rng.choice([0, 0, 0, 1, 130, 1500]),
                "heads": kv * group, "kv_heads": kv, "dim": dim, "dtype": dtype, "bias": rng.choice([0, 0, 1, 40, 128, 500]),
                "layout": layout}
    if op == "append":
        total = _spread(rng, 1, max(1, 16384 * 1024 // (kv * max(dim, 64))))
        return {"op": op, "seqs": min(total, _spread(rng, 1, 128)), "total": total, "past": rng.choice([0, 1, 77, 500]), "kv_heads": kv,
                "dim": dim, "dtype": dtype, "format": fmt, "page": page, "layout": layout}
    if op == "read":
        total = _spread(rng, 1, max(1, 65536 * 1024 // (kv * max(dim, 64))))
        return {"op": op, "seqs": min(total, _spread(rng, 1, 64)), "total": total, "kv_heads": kv, "dim": dim, "dtype": dtype,
                "format": fmt, "page": page, "layout": layout}
    if op == "decode":
        group = rng.choice([1, 2, 4, 7, 8, 16])
        total = _spread(rng, 1, max(1, 262144 * 1024 // (kv * max(dim, 64))))
        return {"op": op, "seqs": min(total, _spread(rng, 1, 128)), "total": total, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "dtype": dtype, "format": fmt, "page": page, "bias": rng.choice([0, 0, 1, 128, 500]), "layout": layout}
    vocab = _spread(rng, 2, 200000)
    return {"op": op, "rows": _spread(rng, 1, max(1, min(512, 256 * 131072 // vocab))), "vocab": vocab,
            "dtype": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "mode": rng.choice(["all", "top_k", "top_p", "min_p", "mixed"]),
            "layout": layout}


def _lengths(case):
    """Uneven lengths that sum to ``total``: half the sequences near the mean, the others anywhere
    from one token up; fixed by the case alone."""
    n, total = case["seqs"], case["total"]
    r = random.Random(case["layout"])
    if case["op"] == "append" and total == n:
        return [1] * n
    share = [r.uniform(0.7, 1.3) if i % 2 else math.exp(r.uniform(-3, 1)) for i in range(n)]
    scale = (total - n) / sum(share)
    lens = [1 + int(s * scale) for s in share]
    lens[r.randrange(n)] += total - sum(lens)
    return lens


def _pages(case, capacity):
    """A table of page numbers in no order, -1 behind each sequence's last page, and the pool's size."""
    page = case["page"]
    need = [-(-c // page) for c in capacity]
    r = random.Random(case["layout"] + 1)
    numbers = list(range(sum(need) + 3))
    r.shuffle(numbers)
    width, rows, at = max(need), [], 0
    for c in need:
        rows.append(numbers[at:at + c] + [-1] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32), len(numbers)


def _cumulative(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32)


def _scales(amax, fmt):
    """fp32 quotients, rounded once (a division by a number becomes a product with its reciprocal)."""
    return (amax / torch.full_like(amax, QMAX[fmt])).clamp_min(2.0 ** -126)


# ---- inputs --------------------------------------------------------------------------------------
def _cache_of(case, pool, g, dev, filled):
    """Codes and scales of a pool of pages; ``filled`` holds values of unit deviation quantised row by row."""
    width = -(-case["dim"] // 16) * 16
    shape = (pool, case["kv_heads"], case["page"], width)
    parts = {}
    for name in ("k", "v"):
        if filled:
            x = torch.randn(shape, generator=g, device=dev)
            x[..., case["dim"]:] = 0
            scale = _scales(x.abs().amax(-1), case["format"])
            q = x / scale[..., None]
            q = q.clamp(-127, 127).round() if case["format"] == "int8" else q.clamp(-448, 448)
            parts[name + "_codes"], parts[name + "_scale"] = q.to(CODE[case["format"]]), scale
        else:
            parts[name + "_codes"] = torch.zeros(shape, dtype=torch.uint8, device=dev).view(CODE[case["format"]])
            parts[name + "_scale"] = torch.zeros(shape[:3], device=dev)
    return parts


def _handle(case, parts, dev):
    """What a user keeps: the framework's cache object, or the bare tensors for the plain form."""
    if not own:
        return parts
    from qmoe_b200 import serving
    cache = serving.QuantCache(parts["k_codes"].shape[0], case["page"], case["kv_heads"], case["dim"], dev,
                               fmt=case["format"])
    for name, value in parts.items():
        getattr(cache, name).view(torch.uint8).copy_(value.view(torch.uint8))
    return cache


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    st = {"case": case}
    op = case["op"]
    if op == "sample":
        n, vocab = case["rows"], case["vocab"]
        logits = torch.randn(n, vocab, generator=g, device=dev) * 2.5
        logits.masked_fill_(torch.rand(n, vocab, generator=g, device=dev) < 0.02, -math.inf)   # banned tokens
        logits[:, 0] = 0.5                                                                      # never a row without any
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        st["u"] = torch.rand(n, generator=g, device=dev)
        mode = case["mode"]
        pick = torch.randint(0, 5, (n,), generator=g, device=dev) if mode == "mixed" else torch.zeros(n, device=dev)
        st["temperature"] = torch.where(pick == 4, torch.zeros(n, device=dev), 0.4 + torch.rand(n, generator=g, device=dev))
        st["top_k"] = torch.randint(1, 100, (n,), generator=g, device=dev, dtype=torch.int32) if mode in ("mixed", "top_k") \
            else torch.zeros(n, dtype=torch.int32, device=dev)
        st["top_k"] = torch.where((pick == 1) | (pick == 2), torch.zeros_like(st["top_k"]), st["top_k"])
        st["top_p"] = 0.5 + 0.5 * torch.rand(n, generator=g, device=dev) if mode in ("mixed", "top_p") else torch.ones(n, device=dev)
        st["min_p"] = 0.1 * torch.rand(n, generator=g, device=dev) if mode in ("mixed", "min_p") else torch.zeros(n, device=dev)
        return st
    lens = _lengths(case)
    hk, d, dt = case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    if case.get("bias"):
        st["bias"] = 0.5 * torch.randn(case["heads"], case["bias"], generator=g, device=dev)
    # unscaled scores (the biased form) meet projections that are small enough for them
    small = d ** -0.25 if case.get("bias") else 1.0
    st["scale"] = 1.0 if case.get("bias") else d ** -0.5
    if op == "prompt":
        # queries, keys and values leave one projection side by side, as the decoder's do
        lens_k = [n + case["prefix"] for n in lens]
        if case["prefix"]:
            kv = torch.randn(sum(lens_k), 2, hk, d, generator=g, device=dev) * torch.tensor([small, 1.0], device=dev)[:, None, None]
            kv = kv.to(dt)
            st["q"] = (torch.randn(case["total"], case["heads"], d, generator=g, device=dev) * small).to(dt)
            st["k"], st["v"] = kv[:, 0], kv[:, 1]
        else:
            rows = torch.randn(case["total"], case["heads"] + 2 * hk, d, generator=g, device=dev)
            rows[:, :case["heads"] + hk] *= small
            rows = rows.to(dt)
            st["q"], st["k"], st["v"] = rows.split([case["heads"], hk, hk], 1)
        st["lens"], st["lens_k"] = lens, lens_k
        st["cu_q"], st["cu_k"] = _cumulative(lens).to(dev), _cumulative(lens_k).to(dev)
        return st
    past = case.get("past", 0)
    table, pool = _pages(case, [n + past for n in lens])
    st["table_host"], st["table"] = table, table.to(dev)
    st["lens"], st["cu"] = lens, _cumulative(lens).to(dev)
    st["start"] = torch.full((len(lens),), past, dtype=torch.int32, device=dev)
    st["parts"] = _cache_of(case, pool, g, dev, filled=op != "append")
    st["cache"] = _handle(case, st["parts"], dev)
    if op == "append":
        kv = torch.randn(case["total"], 2, hk, d, generator=g, device=dev).to(dt)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]
    if op == "decode":
        st["q"] = (torch.randn(len(lens), case["heads"], d, generator=g, device=dev) * small).to(dt)
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    return st


# ---- plain forms ---------------------------------------------------------------------------------
def _plain_attention(q, k, v, scale, bias, first):
    """q [h, n, d], k / v [hk, m, d] in 32 bits; query i of the n sees keys 0 .. first + i."""
    h, n, d = q.shape
    hk, m, _ = k.shape
    group = h // hk
    out = torch.empty_like(q)
    at_once = max(1, (1 << 27) // (m * group * n))                     # key heads whose scores are held together
    rows = n if at_once > 1 else max(1, (1 << 27) // (m * group))
    at_k = torch.arange(m, device=q.device)
    for a in range(0, hk, at_once):
        ks, vs = k[a:a + at_once, None], v[a:a + at_once, None]
        heads = slice(a * group, (a + ks.shape[0]) * group)
        for r in range(0, n, rows):
            qs = q[heads, r:r + rows].unflatten(0, (-1, group))
            s = (qs @ ks.transpose(-1, -2)) * scale
            at_q = torch.arange(r, r + qs.shape[2], device=q.device) + first
            away = at_q[:, None] - at_k[None, :]
            if bias is not None:
                s = s + bias[heads][:, away.clamp(0, bias.shape[1] - 1)].unflatten(0, (-1, group))
            s = s.masked_fill(away < 0, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            o = (p @ vs) / torch.where(total == 0, torch.ones_like(total), total)
            out[heads, r:r + rows] = o.flatten(0, 1)
    return out


def _plain_prompt(st):
    out = torch.empty(st["q"].shape, dtype=st["q"].dtype, device=st["q"].device)
    a = b = 0
    for n, m in zip(st["lens"], st["lens_k"]):
        o = _plain_attention(st["q"][a:a + n].transpose(0, 1).float(), st["k"][b:b + m].transpose(0, 1).float(),
                             st["v"][b:b + m].transpose(0, 1).float(), st["scale"], st.get("bias"), m - n)
        out[a:a + n] = o.transpose(0, 1).to(out.dtype)
        a, b = a + n, b + m
    return out


def _plain_slots(st):
    """Page and place inside it of every row of the packed batch."""
    page = st["case"]["page"]
    dev = st["cu"].device
    n = torch.arange(st["case"]["total"], device=dev)
    seq = torch.searchsorted(st["cu"][1:].long(), n, right=True)
    pos = n - st["cu"].long()[seq] + st["start"].long()[seq]
    return st["table"].long()[seq, pos // page], pos % page


def _plain_codes(x, fmt):
    """(values of the codes in 64 bits, scales in 32): the quotient is rounded once, in 64 bits."""
    scale = _scales(x.float().abs().amax(-1), fmt)
    y = x.double() / scale.double()[..., None]
    if fmt == "int8":
        return y.round().clamp(-127, 127), scale
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return ((y / step).round() * step).clamp(-448, 448), scale


def _plain_append(st):
    parts, case = st["parts"], st["case"]
    at, inside = _plain_slots(st)
    for name in ("k", "v"):
        value, scale = _plain_codes(st[name], case["format"])
        codes = value.float().to(CODE[case["format"]]).view(torch.uint8)
        codes = torch.nn.functional.pad(codes, (0, parts[name + "_codes"].shape[-1] - case["dim"]))
        parts[name + "_codes"].view(torch.uint8)[at, :, inside] = codes
        parts[name + "_scale"][at, :, inside] = scale
    return dict(parts)


def _plain_rows(parts, name, at, inside, dim):
    codes = parts[name + "_codes"]
    values = codes.view(torch.uint8)[at, :, inside].view(codes.dtype).float()[..., :dim]
    return values * parts[name + "_scale"][at, :, inside][..., None]


def _plain_read(st):
    at, inside = _plain_slots(st)
    dt = DTYPES[st["case"]["dtype"]]
    return tuple(_plain_rows(st["parts"], name, at, inside, st["case"]["dim"]).to(dt) for name in ("k", "v"))


def _plain_decode(st):
    case = st["case"]
    out = torch.empty_like(st["q"])
    for i, n in enumerate(st["lens"]):
        pos = torch.arange(n, device=out.device)
        at, inside = st["table"].long()[i, pos // case["page"]], pos % case["page"]
        k, v = (_plain_rows(st["parts"], name, at, inside, case["dim"]).transpose(0, 1) for name in ("k", "v"))
        o = _plain_attention(st["q"][i].float()[:, None], k, v, st["scale"], st.get("bias"), n - 1)
        out[i] = o[:, 0].to(out.dtype)
    return out


def _plain_sample(st):
    x = st["logits"].double()
    n, vocab = x.shape
    top = x.amax(1, keepdim=True)
    index = torch.arange(vocab, device=x.device)
    best = torch.where(x == top, index, vocab).amin(1)
    t = st["temperature"].double()[:, None]
    w = torch.exp((x - top) / torch.where(t == 0, torch.ones_like(t), t))
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    k = st["top_k"].long()[:, None]
    ws = torch.where((k <= 0) | (index < k), ws, torch.zeros_like(ws))
    cum = ws.cumsum(1)
    before = torch.nn.functional.pad(cum[:, :-1], (1, 0))
    p = st["top_p"].double()[:, None]
    ws = torch.where((p >= 1) | (before < p * cum[:, -1:]) | (index == 0), ws, torch.zeros_like(ws))
    ws = torch.where(ws >= st["min_p"].double()[:, None], ws, torch.zeros_like(ws))
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    cum = kept.cumsum(1)
    total = cum[:, -1:]
    token = (cum <= st["u"].double()[:, None] * total).sum(1)
    token = torch.where(t[:, 0] == 0, best, token)
    logprob = torch.log(kept.gather(1, token[:, None]) / total)[:, 0]
    return token, torch.where(t[:, 0] == 0, torch.zeros_like(logprob), logprob).float()


# ---- one pass ------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "read": _plain_read, "decode": _plain_decode,
                "sample": _plain_sample}[op](state)
    from qmoe_b200 import serving
    if op == "prompt":
        return serving.prompt_attention(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"],
                                        scale=state["scale"], rel_bias=state.get("bias"))
    cache = state.get("cache")
    if op == "append":
        serving.cache_append(cache, state["k"], state["v"], state["cu"], state["start"], state["table"])
        return {"k_codes": cache.k_codes, "k_scale": cache.k_scale, "v_codes": cache.v_codes, "v_scale": cache.v_scale}
    if op == "read":
        return serving.cache_read(cache, state["cu"], state["start"], state["table"], state["case"]["total"],
                                  dtype=DTYPES[state["case"]["dtype"]])
    if op == "decode":
        return serving.decode_attention_paged(state["q"], cache, state["table"], state["lengths"], scale=state["scale"],
                                              rel_bias=state.get("bias"))
    return serving.sample_tokens(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"], return_logprob=True)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "sample":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["rows"]
        # an exponential and a sum for every logit
        return {"bytes": n * case["vocab"] * size + n * (5 * 4 + 8 + 4), "flops": 2 * n * case["vocab"]}
    lens = _lengths(case)
    d, hk = case["dim"], case["kv_heads"]
    if op == "prompt":
        pairs = sum(n * (case["prefix"] + 1) + n * (n - 1) // 2 for n in lens)
        rows_k = case["total"] + case["prefix"] * len(lens)
        return {"bytes": 2 * d * (2 * case["total"] * case["heads"] + 2 * rows_k * hk) + 4 * case["heads"] * case["bias"],
                "flops": 4 * pairs * case["heads"] * d}
    rows = case["total"] * hk
    if op in ("append", "read"):
        return {"bytes": 2 * rows * (2 * d + d + 4), "flops": 2 * rows * d}
    return {"bytes": 2 * rows * (d + 4) + 2 * 2 * len(lens) * case["heads"] * d + 4 * case["heads"] * case["bias"],
            "flops": 4 * case["total"] * case["heads"] * d}


# ---- 64 bits -------------------------------------------------------------------------------------
def _exact_attend(q, k, v, scale, bias, offset):
    """One head in 64 bits, by blocks of queries: q [n, d], k / v [m, d], bias [x] or None."""
    n, m = q.shape[0], k.shape[0]
    out = torch.zeros_like(q)
    block = max(1, (1 << 26) // max(m, 1))
    for lo in range(0, n, block):
        hi = min(n, lo + block)
        seen = min(m, offset + hi)                     # keys that the block's last query sees
        if seen <= 0:
            continue
        dist = (offset + torch.arange(lo, hi, device=q.device)).unsqueeze(1) - torch.arange(seen, device=q.device)
        logit = torch.einsum("nd,md->nm", q[lo:hi], k[:seen]) * scale
        if bias is not None:
            logit += bias[torch.minimum(dist.clamp_min(0), torch.tensor(bias.numel() - 1, device=q.device))]
        logit[dist < 0] = -math.inf
        weight = torch.softmax(logit, 1)
        out[lo:hi] = torch.nan_to_num(weight, nan=0.0) @ v[:seen]
    return out


def _exact_places(case, table):
    """[(sequence, first row, page numbers, places)] of a case's packed rows."""
    past, first, found = case.get("past", 0), 0, []
    for s, n in enumerate(_lengths(case)):
        pos = torch.arange(past, past + n)
        found.append((s, first, table[s].long()[torch.div(pos, case["page"], rounding_mode="floor")], pos % case["page"]))
        first += n
    return found


def _exact_codes(x, fmt):
    """Nearest code of x / scale, ties to the even code, found among the sorted values of all codes."""
    scale = torch.clamp((x.abs().amax(-1) / QMAX[fmt]).float(), min=2.0 ** -126)
    if fmt == "int8":
        values = torch.arange(-127, 128, dtype=torch.float64, device=x.device)
        even = torch.arange(-127, 128, device=x.device) % 2 == 0
    else:
        low = [m / 8 * 2.0 ** -6 for m in range(8)]
        high = [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1]     # the last one is NaN
        pos = low + high
        values = torch.tensor([-a for a in reversed(pos[1:])] + pos, dtype=torch.float64, device=x.device)
        code = list(range(len(pos)))
        even = torch.tensor([c % 2 == 0 for c in list(reversed(code[1:])) + code], device=x.device)
    y = x / scale.double().unsqueeze(-1)
    above = torch.searchsorted(values, y.contiguous()).clamp(1, values.numel() - 1)
    below = above - 1
    up, down = values[above] - y, y - values[below]
    take_up = (up < down) | ((up == down) & even[above])
    return torch.where(take_up, values[above], values[below]), scale


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "prompt":
        q, k, v = st["q"].double(), st["k"].double(), st["v"].double()
        out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
        group = case["heads"] // case["kv_heads"]
        a = b = 0
        for n in _lengths(case):
            m = n + case["prefix"]
            for h in range(case["heads"]):
                bias = st["bias"][h].double() if "bias" in st else None
                out[a:a + n, h] = _exact_attend(q[a:a + n, h], k[b:b + m, h // group], v[b:b + m, h // group], st["scale"], bias, m - n)
            a, b = a + n, b + m
        return out
    if op == "sample":
        return _exact_sample(st)
    places = _exact_places(case, st["table_host"])
    parts, d = st["parts"], case["dim"]
    if op == "append":
        result = {}
        for name in ("k", "v"):
            codes = parts[name + "_codes"].float().double()
            scales = parts[name + "_scale"].double()
            value, scale = _exact_codes(st[name].double(), case["format"])
            for s, first, at, inside in places:
                n = at.numel()
                codes[at.to(codes.device), :, inside.to(codes.device), :d] = value[first:first + n]
                scales[at.to(codes.device), :, inside.to(codes.device)] = scale[first:first + n].double()
            result[name + "_codes"], result[name + "_scale"] = codes, scales
        if case["format"] == "int8":
            for name in ("k_codes", "v_codes"):
                result[name] = result[name].to(torch.int8)
        return {"k_codes": result["k_codes"], "k_scale": result["k_scale"], "v_codes": result["v_codes"],
                "v_scale": result["v_scale"]}

    def rows(name, at, inside):
        at, inside = at.to(st["cu"].device), inside.to(st["cu"].device)
        codes = parts[name + "_codes"].view(torch.uint8)[at, :, inside].view(CODE[case["format"]])
        return codes.float().double()[..., :d] * parts[name + "_scale"][at, :, inside].double().unsqueeze(-1)

    if op == "read":
        return tuple(torch.cat([rows(name, at, inside) for _, _, at, inside in places]) for name in ("k", "v"))
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    group = case["heads"] // case["kv_heads"]
    for s, _, at, inside in places:
        k, v = rows("k", at, inside), rows("v", at, inside)
        n = k.shape[0]
        q = st["q"][s].double().reshape(case["kv_heads"], group, d)
        logit = torch.einsum("agd,nad->agn", q, k) * st["scale"]
        if "bias" in st:
            back = torch.arange(n - 1, -1, -1, device=out.device).clamp_max(case["bias"] - 1)
            logit += st["bias"].double()[:, back].reshape(case["kv_heads"], group, n)
        out[s] = torch.einsum("agn,nad->agd", torch.softmax(logit, -1), v).reshape(case["heads"], d)
    return out


def _exact_sample(st):
    """Row by row, from the sorted list downwards."""
    logits = st["logits"].double()
    tokens, logprobs = [], []
    settings = zip(*(st[name].tolist() for name in ("temperature", "top_k", "top_p", "min_p", "u")))
    for row, (t, k, p, least, u) in zip(logits, settings):
        if t == 0:
            tokens.append(torch.nonzero(row == row.max())[0, 0])
            logprobs.append(torch.zeros((), dtype=torch.float64, device=row.device))
            continue
        value, where = torch.sort(row, dim=0, descending=True, stable=True)
        if k > 0:
            value, where = value[:k], where[:k]
        share = torch.softmax(value / t, 0)
        count = value.numel()
        if p < 1:
            upto = torch.cumsum(share, 0) - share
            count = max(1, int((upto < p).sum()))
        count = min(count, max(1, int((torch.exp((value - value[0]) / t) >= least).sum())))
        by_index, back = torch.sort(where[:count])
        mass = torch.exp((value[:count] - value[0]) / t)[back]
        total = torch.cumsum(mass, 0)
        at = int((total <= u * total[-1]).sum())
        tokens.append(by_index[at])
        logprobs.append(torch.log(mass[at] / total[-1]))
    return torch.stack(tokens), torch.stack(logprobs)
