"""The operators of batched serving, as cases that can be timed and whose outputs can be compared.

Four operators that a server of several sequences runs between its quantized linears, through the public entry points
(`nanoserve_b200.ops.Kernels`):
  append   `paged_kv_append`: bias and rotary embedding on a batch's q | k | v rows, k and v into the pages of a cache
  attend   `paged_attention`: new tokens (one each, or chunks of prompts) against the paged cache, causal, with a sliding
           window and first tokens that stay visible
  prefix   `shared_prefix_attention`: one new token per sequence, all sequences behind one long prefix that is stored once
  sample   `sample`: tokens from logits by temperature, top-k, top-p and min-p, with given random numbers
Head layouts are those of the 7B- and 70B-class layers (28 and 4 heads, 64 and 8 heads of 128) and generic ones; the
vocabulary is the runner's.  `own` chooses between the framework's calls and a plain form of the same operators.
"""
import math
import random

import numpy as np
import torch

own = False

# the largest listed work, which no drawn case exceeds: scores of the plain form, elements of keys, logits, appended rows
MOST_SCORES = 28 * 8192 * 8192
MOST_KEYS = 16 * 32768 * 4 * 128
MOST_PREFIX_SCORES = 64 * 28 * (32771 + 2000)
MOST_LOGITS = 64 * 152064
MOST_ROWS = 8192 * 36 * 128

_kernels = None


def kernels():
    global _kernels
    if _kernels is None:
        from nanoserve_b200.ops import Kernels
        _kernels = Kernels()
        _kernels.init()
    return _kernels


def listed():
    heads = dict(n_heads=28, n_kv_heads=4, head_dim=128)
    return [
        # one decode step of a small batch: a new row per sequence, the smallest call
        dict(name="append_tokens_16", op="append", n_seqs=16, new_lo=1, new_hi=1, past_lo=40, past_hi=4000, page=16, bias=True,
             lens_seed=1, **heads),
        # prompts of several requests in one batch, some on top of earlier turns
        dict(name="append_prompts_8k", op="append", n_seqs=5, new_lo=1021, new_hi=2200, past_lo=0, past_hi=30000, page=64,
             bias=True, lens_seed=2, **heads),
        # single-stream decode behind a short conversation: latency
        dict(name="attend_token_1", op="attend", n_seqs=1, new_lo=1, new_hi=1, past_lo=700, past_hi=700, page=16, window=512,
             sinks=4, lens_seed=3, **heads),
        # a decode batch of ragged lengths with a long window
        dict(name="attend_tokens_16", op="attend", n_seqs=16, new_lo=1, new_hi=1, past_lo=500, past_hi=32767, page=64,
             window=4096, sinks=4, lens_seed=4, **heads),
        # chunks of prompts behind what is cached, a small model's heads
        dict(name="attend_chunks_3", op="attend", n_seqs=3, new_lo=150, new_hi=517, past_lo=300, past_hi=5000, page=32,
             window=1024, sinks=4, lens_seed=5, n_heads=16, n_kv_heads=2, head_dim=64),
        # a long prompt at once: the largest matrix work
        dict(name="attend_prompt_8k", op="attend", n_seqs=1, new_lo=8192, new_hi=8192, past_lo=0, past_hi=0, page=128,
             window=4096, sinks=4, lens_seed=6, **heads),
        # three continuations of a short common instruction
        dict(name="prefix_3", op="prefix", n_seqs=3, prefix=777, own_lo=1, own_hi=200, page=16, lens_seed=7, **heads),
        # a decode batch behind a system prompt
        dict(name="prefix_16", op="prefix", n_seqs=16, prefix=8192, own_lo=16, own_hi=512, page=64, lens_seed=8, **heads),
        # many samples of one long document, odd length
        dict(name="prefix_64", op="prefix", n_seqs=64, prefix=32771, own_lo=100, own_hi=2000, page=128, lens_seed=9, **heads),
        # the pick of a single stream's next token
        dict(name="sample_1", op="sample", n_seqs=1, vocab=152064, dtype="bfloat16", filters="kp"),
        # a decode batch with top-p alone: no small set to look at
        dict(name="sample_16", op="sample", n_seqs=16, vocab=152064, dtype="bfloat16", filters="p"),
        # a large batch, each row with its own settings, logits in 32 bits
        dict(name="sample_64", op="sample", n_seqs=64, vocab=152064, dtype="float32", filters="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix", "sample"])
    if op == "sample":
        V = rng.choice([152064, _log_int(rng, 1000, 152064)])
        B = min(_log_int(rng, 1, 64), MOST_LOGITS // V)
        return dict(op=op, n_seqs=B, vocab=V, dtype=rng.choice(["bfloat16", "float32"]),
                    filters=rng.choice(["kp", "p", "mixed", "none"]))
    Hq, Hk, D = rng.choice([(28, 4, 128), (28, 4, 128), (64, 8, 128), (16, 2, 64), (8, 8, 64), (32, 8, 128)])
    heads = dict(n_heads=Hq, n_kv_heads=Hk, head_dim=D, page=rng.choice([16, 32, 64, 128, 256]), lens_seed=rng.randrange(1 << 30))
    while True:
        B = _log_int(rng, 1, 64)
        if op == "append":
            new = _log_int(rng, 1, 4096)
            case = dict(op=op, n_seqs=B, new_lo=(new + 1) // 2, new_hi=new, past_lo=0, past_hi=_log_int(rng, 1, 8000),
                        bias=rng.random() < 0.7, **heads)
            if B * new * (Hq + 2 * Hk) * D <= MOST_ROWS and B * (new + case["past_hi"]) * Hk * D <= MOST_KEYS:
                return case
        elif op == "attend":
            new = rng.choice([1, 1, _log_int(rng, 1, 16), _log_int(rng, 16, 8192)])
            past = _log_int(rng, 1, 32768)
            case = dict(op=op, n_seqs=B, new_lo=(new + 1) // 2, new_hi=new, past_lo=past // 8, past_hi=past,
                        window=rng.choice([0, _log_int(rng, 16, 8192)]), sinks=rng.choice([0, 1, 4, 64]), **heads)
            if B * Hq * new * (new + past) <= MOST_SCORES and B * (new + past) * Hk * D <= MOST_KEYS:
                return case
        else:
            own_hi = _log_int(rng, 1, 2000)
            case = dict(op=op, n_seqs=B, prefix=_log_int(rng, 16, 32771), own_lo=(own_hi + 7) // 8, own_hi=own_hi, **heads)
            if B * Hq * (case["prefix"] + own_hi) <= MOST_PREFIX_SCORES and B * own_hi * Hk * D <= MOST_KEYS:
                return case


def lengths(case):
    """New and cached tokens of every sequence, fixed by the case."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "prefix":
        return [1] * case["n_seqs"], [rng.randint(case["own_lo"], case["own_hi"]) for _ in range(case["n_seqs"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n_seqs"])]
    past = [_log_int(rng, case["past_lo"] + 1, case["past_hi"] + 1) - 1 for _ in range(case["n_seqs"])]
    return new, [n + p for n, p in zip(new, past)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)
    st = {"case": case}
    B = case["n_seqs"]
    if case["op"] == "sample":
        # a language model's logits: a few likely tokens, then a power law over the rest, in an order of their own per row
        V, filters = case["vocab"], case["filters"]
        order = torch.argsort(rand(B, V), dim=-1)
        fall = -(1.0 + 0.6 * rand(B, 1)) * torch.log(torch.arange(1, V + 1, device="cuda").float())
        logits = torch.zeros(B, V, device="cuda").scatter_(1, order, fall + 0.3 * randn(B, V)) + 14.0
        st["logits"] = logits.to(getattr(torch, case["dtype"]))
        st["u"] = rand(B)
        pick = lambda *choices: torch.tensor(choices, device="cuda")[torch.randint(len(choices), (B,), device="cuda",
                                                                                     generator=gen)]
        st["temperature"] = 0.6 + 0.6 * rand(B)
        st["top_k"] = pick(50, 50, 200, 20) if filters == "kp" else pick(0, 0, 20, 50, 1000) if filters == "mixed" else pick(0)
        st["top_p"] = pick(1.0) if filters == "none" else pick(0.9, 0.95) if filters != "mixed" else pick(1.0, 0.95, 0.9, 0.5)
        st["min_p"] = pick(0.0, 0.02, 0.1) if filters == "mixed" else pick(0.0)
        st["top_k"] = st["top_k"].to(torch.int32)
        return st
    new, lens = lengths(case)
    Hq, Hk, D, page = case["n_heads"], case["n_kv_heads"], case["head_dim"], case["page"]
    T = sum(new)
    prefix = case.get("prefix", 0)
    n_prefix = -(-prefix // page)
    width = max(-(-n // page) for n in lens)
    n_pages = n_prefix + sum(-(-n // page) for n in lens) + 3
    ids = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32)  # pages are given out in no order
    table = torch.zeros(B, width, dtype=torch.int32)
    at = n_prefix + torch.cumsum(torch.tensor([0] + [-(-n // page) for n in lens]), 0)
    col = torch.arange(width)
    st["block_table"] = ids[(at[:-1, None] + torch.minimum(col[None], (at[1:] - at[:-1])[:, None] - 1)).to("cuda").long()].contiguous()
    st["prefix_table"] = ids[:n_prefix].contiguous()
    st["prefix_len"] = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["cu_tokens"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    st["max_new"], st["max_len"] = max(new), max(lens)
    # which sequence a row belongs to, its place among the sequence's new tokens and in the sequence
    seq = np.repeat(np.arange(B), new)
    nth = np.concatenate([np.arange(n) for n in new])
    st["seq"], st["nth"] = (torch.tensor(a, device="cuda") for a in (seq, nth))
    st["position"] = torch.tensor(nth + np.repeat(np.array(lens) - np.array(new), new), device="cuda")
    kv = lambda: torch.empty(n_pages, Hk, page, D, dtype=torch.bfloat16, device="cuda")
    st["cache_k"], st["cache_v"] = kv().normal_(generator=gen), kv().normal_(generator=gen)
    if case["op"] == "append":
        st["qkv"] = randn(T, (Hq + 2 * Hk) * D).to(torch.bfloat16)
        st["bias"] = (0.3 * randn((Hq + 2 * Hk) * D)).to(torch.bfloat16) if case["bias"] else None
        st["inv_freq"] = 1.0 / (1e6 ** (torch.arange(0, D, 2, device="cuda").float() / D))
    else:
        st["q"] = (1.5 * randn(T, Hq * D)).to(torch.bfloat16)
    return st


# ---- the plain form

def _plain_append(st):
    c = st["case"]
    Hq, Hk, D, page = c["n_heads"], c["n_kv_heads"], c["head_dim"], c["page"]
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = x + st["bias"].float()
    x = x.view(x.shape[0], Hq + 2 * Hk, D)
    angle = st["position"].double()[:, None] * st["inv_freq"].double()[None]  # far positions: 32 bits lose the angle
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    lo, hi = x[:, :Hq + Hk, :D // 2], x[:, :Hq + Hk, D // 2:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(torch.bfloat16)
    pages = st["block_table"][st["seq"], st["position"] // page].long()
    st["cache_k"][pages, :, st["position"] % page] = rot[:, Hq:]
    st["cache_v"][pages, :, st["position"] % page] = x[:, Hq + Hk:].to(torch.bfloat16)
    return {"q": rot[:, :Hq].reshape(-1, Hq * D), "cache_k": st["cache_k"], "cache_v": st["cache_v"]}


def _gathered(cache, table, n, page):
    """Rows 0 .. n - 1 of every sequence of a table: [B, Hk, n, D] in 32 bits."""
    at = torch.arange(n, device=cache.device)
    return cache[table[:, at // page].long(), :, (at % page)[None]].permute(0, 2, 1, 3).float()


def _plain_attend(st):
    c = st["case"]
    Hq, Hk, D, page, B = c["n_heads"], c["n_kv_heads"], c["head_dim"], c["page"], c["n_seqs"]
    M, L, g = st["max_new"], st["max_len"], c["n_heads"] // c["n_kv_heads"]
    k = _gathered(st["cache_k"], st["block_table"], L, page)
    v = _gathered(st["cache_v"], st["block_table"], L, page)
    q = torch.zeros(B, M, Hq, D, device=k.device)
    q[st["seq"], st["nth"]] = st["q"].view(-1, Hq, D).float()
    q = q.view(B, M, Hk, g, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, g * M, D)
    s = (q @ k.transpose(-1, -2) / math.sqrt(D)).view(B, Hk, g, M, L)
    n_new = st["cu_tokens"][1:] - st["cu_tokens"][:-1]
    pos = (st["seq_lens"] - n_new)[:, None] + torch.arange(M, device=k.device)[None]  # [B, M]
    j = torch.arange(L, device=k.device)
    seen = j <= pos[..., None]
    if c["window"]:
        seen &= (j > pos[..., None] - c["window"]) | (j < c["sinks"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, Hk, g * M, L) @ v).view(B, Hk, g, M, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, M, Hq * D)
    return o[st["seq"], st["nth"]].to(torch.bfloat16)


def _plain_prefix(st):
    c = st["case"]
    Hq, Hk, D, page, B, P = c["n_heads"], c["n_kv_heads"], c["head_dim"], c["page"], c["n_seqs"], c["prefix"]
    L, g = st["max_len"], c["n_heads"] // c["n_kv_heads"]
    q = st["q"].view(B, Hk, g, D).float()
    k = _gathered(st["cache_k"], st["prefix_table"][None], P, page)[0]
    s_pre = (q.transpose(0, 1).reshape(Hk, B * g, D) @ k.transpose(-1, -2)).view(Hk, B, g, P).transpose(0, 1)
    s_own = q @ _gathered(st["cache_k"], st["block_table"], L, page).transpose(-1, -2)
    s_own = s_own.masked_fill(torch.arange(L, device=q.device) >= st["seq_lens"][:, None, None, None], -math.inf)
    s = torch.cat([s_pre, s_own], -1) / math.sqrt(D)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = _gathered(st["cache_v"], st["prefix_table"][None], P, page)[0]
    o = (p[..., :P].transpose(0, 1).reshape(Hk, B * g, P) @ v).view(Hk, B, g, D).transpose(0, 1)
    o = o + p[..., P:] @ _gathered(st["cache_v"], st["block_table"], L, page)
    return o.reshape(B, Hq * D).to(torch.bfloat16)


def _plain_sample(st):
    x = st["logits"].double()  # long sums, and values next to a border: 64 bits
    V = x.shape[1]
    w = torch.exp((x - x.amax(-1, keepdim=True)) / st["temperature"].double()[:, None])
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices  # equal logits: the lowest index first
    rank = torch.arange(V, device=x.device)
    k = st["top_k"][:, None]
    ws = w.gather(1, order)
    ws = ws * ((rank < k) | (k <= 0)) * (ws >= st["min_p"].double()[:, None])
    before = torch.cumsum(ws, -1) - ws
    p = st["top_p"].double()[:, None]
    ws = ws * ((before < p * ws.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0))
    cum = torch.cumsum(torch.zeros_like(w).scatter_(1, order, ws), -1)
    return (cum > st["u"].double()[:, None] * cum[:, -1:]).to(torch.uint8).argmax(-1)


def run(st):
    c = st["case"]
    if own:
        k = kernels()
        if c["op"] == "sample":
            return k.sample(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                            min_p=st["min_p"])
        heads = (c["n_heads"], c["n_kv_heads"], c["head_dim"])
        cu = None if st["max_new"] == 1 else st["cu_tokens"]
        if c["op"] == "append":
            q = k.paged_kv_append(st["qkv"], st["bias"], st["inv_freq"], st["cache_k"], st["cache_v"], st["block_table"],
                                  st["seq_lens"], *heads, cu_tokens=cu)
            return {"q": q, "cache_k": st["cache_k"], "cache_v": st["cache_v"]}
        if c["op"] == "attend":
            return k.paged_attention(st["q"], st["cache_k"], st["cache_v"], st["block_table"], st["seq_lens"], *heads,
                                     cu_tokens=cu, max_tokens=st["max_new"], window=c["window"], sinks=c["sinks"])
        return k.shared_prefix_attention(st["q"], st["cache_k"], st["cache_v"], st["prefix_table"], st["prefix_len"],
                                         st["block_table"], st["seq_lens"], *heads)
    return {"append": _plain_append, "attend": _plain_attend, "prefix": _plain_prefix, "sample": _plain_sample}[c["op"]](st)


def _visible(case):
    """Pairs of a new token and a key that it sees, and keys that some new token of their sequence sees."""
    new, lens = lengths(case)
    pairs = keys = 0
    for n, length in zip(new, lens):
        at = np.arange(length - n, length)
        if case["window"]:
            first = np.maximum(at - case["window"] + 1, 0)
            pairs += int((at + 1 - first + np.minimum(first, case["sinks"])).sum())
            keys += length - int(first[0]) + min(int(first[0]), case["sinks"])
        else:
            pairs += int((at + 1).sum())
            keys += length
    return pairs, keys


def work(case):
    if case["op"] == "sample":
        n = case["n_seqs"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bfloat16" else 4) + 32 * case["n_seqs"], "flops": 2 * n}
    new, lens = lengths(case)
    Hq, Hk, D, T = case["n_heads"], case["n_kv_heads"], case["head_dim"], sum(new)
    if case["op"] == "append":
        rows = T * (Hq + 2 * Hk) * D
        return {"bytes": 2 * rows * 2 + (Hq + 2 * Hk) * D * 2 * case["bias"] + 2 * D, "flops": 3 * T * (Hq + Hk) * D}
    pairs, keys = _visible(case) if case["op"] == "attend" else (T * case["prefix"] + sum(lens), case["prefix"] + sum(lens))
    return {"bytes": 2 * keys * Hk * D * 2 + 2 * T * Hq * D * 2, "flops": 4 * pairs * Hq * D}


# ---- the operators' definitions in 64 bits, one sequence (or row) after the other

def _sequence(cache, table, n, page):
    pages = table[:-(-n // page)].long()
    return cache[pages].transpose(0, 1).reshape(cache.shape[1], -1, cache.shape[3])[:, :n].double()


def _exact_attend(q, k, v, first, window, sinks):
    """q [n, Hq, D] at positions first, first + 1, ... against keys 0 .. of k, v [Hk, L, D]; a block of rows at a time."""
    n, Hq, D = q.shape
    g = Hq // k.shape[0]
    out = torch.empty_like(q)
    j = torch.arange(k.shape[1], device=q.device)
    for h in range(Hq):
        for i in range(0, n, 2048):
            at = first + torch.arange(i, min(n, i + 2048), device=q.device)[:, None]
            hidden = j[None] > at
            if window:
                hidden = hidden | ((at - j[None] >= window) & (j[None] >= sinks))
            e = torch.einsum("id,jd->ij", q[i:i + 2048, h], k[h // g]) * D ** -0.5
            out[i:i + 2048, h] = torch.softmax(torch.where(hidden, -torch.inf, e), -1) @ v[h // g]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        x = st["logits"].double().cpu().numpy()
        u, t, k, p, m = (st[n].double().cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p"))
        out = np.zeros(len(x), np.int64)
        for b, row in enumerate(x):
            by = np.lexsort((np.arange(row.size), -row))
            w = np.exp((row[by] - row.max()) / t[b])
            n = int(np.sum(w >= m[b]))
            n = n if k[b] <= 0 else min(n, int(k[b]))
            before = np.concatenate([[0.0], np.cumsum(w[:n])])
            if p[b] < 1:
                n = max(1, int(np.searchsorted(before[:n], p[b] * before[n], side="left")))
            kept = np.sort(by[:n])
            cum = np.cumsum(np.exp((row[kept] - row.max()) / t[b]))
            out[b] = kept[np.searchsorted(cum, u[b] * cum[-1], side="right")]
        return torch.from_numpy(out).cuda()
    new, lens = lengths(case)
    Hq, Hk, D, page = case["n_heads"], case["n_kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "append":
        x = st["qkv"].double() + (0 if st["bias"] is None else st["bias"].double())
        z = x.view(-1, Hq + 2 * Hk, 2, D // 2)
        turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                           torch.outer(st["position"].double(), st["inv_freq"].double()))[:, None]
        z = torch.cat([torch.view_as_real(torch.complex(z[:, :Hq + Hk, 0].contiguous(), z[:, :Hq + Hk, 1].contiguous()) * turn)
                       .movedim(-1, -2), z[:, Hq + Hk:]], 1).reshape(-1, Hq + 2 * Hk, D)
        ck, cv = st["cache_k"].double(), st["cache_v"].double()
        slot = st["position"] % page
        to = st["block_table"].long()[st["seq"], torch.div(st["position"], page, rounding_mode="floor")]
        for h in range(Hk):
            ck[to, h, slot] = z[:, Hq + h]
            cv[to, h, slot] = z[:, Hq + Hk + h]
        return {"q": z[:, :Hq].reshape(-1, Hq * D), "cache_k": ck, "cache_v": cv}
    q = st["q"].double().view(-1, Hq, D)
    out, row = torch.empty_like(q), 0
    if case["op"] == "prefix":
        pk, pv = (_sequence(st[c], st["prefix_table"], case["prefix"], page) for c in ("cache_k", "cache_v"))
    for b, (n, length) in enumerate(zip(new, lens)):
        k, v = (_sequence(st[c], st["block_table"][b], length, page) for c in ("cache_k", "cache_v"))
        if case["op"] == "prefix":
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        out[row:row + n] = _exact_attend(q[row:row + n], k, v, k.shape[1] - n, case.get("window", 0), case.get("sinks", 0))
        row += n
    return out.view(-1, Hq * D)
