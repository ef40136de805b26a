"""Timing cases of attention over packed sequences and over a paged cache: dense attention of
sequences of different lengths that lie one after the other (causal or not, grouped heads, with its
gradients), the append of keys and values to a paged cache with the rotary positions applied on the
way, and the attention of a few new tokens over that cache.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes
a case's inputs on the GPU from a seed, ``run()`` makes one pass -- in elementary torch
operations, or with the framework's kernels where ``own`` is true -- ``work()`` counts the
bytes and operations that a pass cannot do without, and ``exact()`` evaluates the same
definitions in 64 bits.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCORES = 1 << 28    # scores that the plain form holds at a time
BASE = 10000.0      # of the rotary frequencies


# ------------------------------------------------------------------------ cases
# "longest", "sequences", "sizes": the lengths, see _lengths.  "keys" of a packed case: "same" (a prompt),
# "more" (a prompt's next part: `before` cached keys at most in front of the queries) or "other"
# (cross-attention to sequences of up to `before` tokens).  "before" of a cache case: tokens already there.
def listed():
    return [
        # a clip's 125 audio tokens at the audio width (1536): latency
        {"name": "packed_audio_clip", "op": "packed", "mode": "fwd", "type": "bf16", "sequences": 1, "longest": 125,
         "sizes": 1, "keys": "same", "before": 0, "causal": False, "hq": 12, "hk": 12, "dim": 128},
        # a batch of prompts of different lengths, 4 query heads a key head
        {"name": "packed_prompts", "op": "packed", "mode": "fwd", "type": "bf16", "sequences": 16, "longest": 2048,
         "sizes": 2, "keys": "same", "before": 0, "causal": True, "hq": 32, "hk": 8, "dim": 128},
        # one long prompt
        {"name": "packed_long_prompt", "op": "packed", "mode": "fwd", "type": "bf16", "sequences": 1, "longest": 32768,
         "sizes": 3, "keys": "same", "before": 0, "causal": True, "hq": 32, "hk": 8, "dim": 128},
        # the next part of four prompts, behind up to 8000 tokens that are there already
        {"name": "packed_next_part", "op": "packed", "mode": "fwd", "type": "fp16", "sequences": 4, "longest": 512,
         "sizes": 4, "keys": "more", "before": 8000, "causal": True, "hq": 40, "hk": 8, "dim": 128},
        # the 720p grid of the 40-head layer attends a text of up to 512 tokens, in training
        {"name": "packed_cross_720p", "op": "packed", "mode": "train", "type": "bf16", "sequences": 1, "longest": 75600,
         "sizes": 5, "keys": "other", "before": 512, "causal": False, "hq": 40, "hk": 40, "dim": 128},
        # training on ragged sequences, odd lengths, 64-wide heads, 6 query heads a key head
        {"name": "packed_train_ragged", "op": "packed", "mode": "train", "type": "bf16", "sequences": 9, "longest": 4093,
         "sizes": 6, "keys": "same", "before": 0, "causal": True, "hq": 24, "hk": 4, "dim": 64},
        # one token of 16 sequences goes to the cache: latency
        {"name": "append_token", "op": "append", "type": "bf16", "sequences": 16, "longest": 1, "sizes": 7,
         "before": 4096, "hq": 32, "hk": 8, "dim": 128, "rot": 128, "layout": "half", "page": 16},
        # whole prompts go to the cache, three quarters of each head rotated
        {"name": "append_prompts", "op": "append", "type": "bf16", "sequences": 16, "longest": 4093, "sizes": 8,
         "before": 0, "hq": 24, "hk": 8, "dim": 128, "rot": 96, "layout": "interleaved", "page": 64},
        # a few sequences that have just begun: latency
        {"name": "paged_begun", "op": "paged", "type": "bf16", "sequences": 4, "new": 1, "longest": 100, "sizes": 9,
         "hq": 32, "hk": 8, "dim": 128, "page": 16},
        # one token of one sequence, far into a long context
        {"name": "paged_long", "op": "paged", "type": "bf16", "sequences": 1, "new": 1, "longest": 131001, "sizes": 10,
         "hq": 32, "hk": 8, "dim": 128, "page": 64},
        # one token each of 64 sequences of different lengths
        {"name": "paged_batch", "op": "paged", "type": "bf16", "sequences": 64, "new": 1, "longest": 4096, "sizes": 11,
         "hq": 32, "hk": 8, "dim": 128, "page": 16},
        # four drafted tokens of 8 sequences, a key head a query head, pages of 100 tokens
        {"name": "paged_draft", "op": "paged", "type": "fp16", "sequences": 8, "new": 4, "longest": 2000, "sizes": 12,
         "hq": 24, "hk": 24, "dim": 64, "page": 100},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        # a pass costs no more than the largest listed ones; caches fit next to each other
        if w["flops"] <= 8e12 and w["bytes"] <= 1.5e9 and _cache_bytes(case) <= 1.1e9:
            return case


def _draw(rng):
    op = rng.choice(["packed", "packed", "append", "paged", "paged"])
    dim, kind, sizes = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "fp16"]), rng.randrange(1 << 20)
    hk = rng.choice([1, 2, 4, 8, 12])
    hq = hk * rng.choice([1, 1, 2, 3, 4, 5, 8])
    sequences = _log(rng, 1, 64)
    if op == "packed":
        mode, keys = rng.choice(["fwd", "train"]), rng.choice(["same", "same", "more", "other"])
        return {"op": op, "mode": mode, "type": "bf16" if mode == "train" else kind, "sequences": sequences,
                "longest": _log(rng, 1, 16384), "sizes": sizes, "keys": keys,
                "before": 0 if keys == "same" else _log(rng, 1, 8192),
                "causal": keys == "more" or (keys == "same" and rng.random() < 0.7), "hq": hq, "hk": hk, "dim": dim}
    page = rng.choice([8, 16, 32, 64, 100, 256])
    if op == "append":
        return {"op": op, "type": kind, "sequences": sequences, "longest": rng.choice([1, _log(rng, 1, 8192)]),
                "sizes": sizes, "before": rng.choice([0, _log(rng, 1, 131072)]), "hq": hq, "hk": hk, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, dim // 4 * 3]), "layout": rng.choice(["interleaved", "half"]),
                "page": page}
    return {"op": op, "type": kind, "sequences": sequences, "new": rng.choice([1, 1, 1, 2, 4, 7]),
            "longest": _log(rng, 8, 131072), "sizes": sizes, "hq": hq, "hk": hk, "dim": dim, "page": page}


def _lengths(case):
    """(tokens of each sequence in this pass, its keys in all)."""
    rng = random.Random(case["sizes"])

    def some(longest):   # the first sequence is the longest
        return [longest] + [_log(rng, max(1, longest // 16), longest) for _ in range(case["sequences"] - 1)]

    if case["op"] == "paged":
        new = case["new"]
        return [new] * case["sequences"], [max(new, n) for n in some(case["longest"])]
    q = some(case["longest"])
    if case["before"] == 0:
        return q, q
    before = some(case["before"])
    return (q, before) if case.get("keys") == "other" else (q, [a + b for a, b in zip(q, before)])


def _pages(case):
    """Pages of each sequence, and of the cache, which has a few that nobody uses."""
    each = [-(-n // case["page"]) for n in _lengths(case)[1]]
    return each, sum(each) + 3


def _cache_bytes(case):
    return 0 if case["op"] == "packed" else 4 * _pages(case)[1] * case["page"] * case["hk"] * case["dim"]


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ----------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]

    def rnd(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    s = dict(case)
    s["q_len"], s["k_len"] = _lengths(case)
    hq, hk, dim, tokens = case["hq"], case["hk"], case["dim"], sum(s["q_len"])
    offsets = torch.tensor(_starts(s["q_len"]), dtype=torch.int32, device="cuda")
    if case["op"] == "packed":
        if s["k_len"] == s["q_len"]:   # slices of a fused projection's output
            qkv = rnd(tokens, hq + 2 * hk, dim)
            s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
            s["q"].mul_(1.5)           # scores of more than unit variance: some keys matter more than others
            s["offsets"], s["k_offsets"] = offsets, None
        else:
            s["q"] = rnd(tokens, hq, dim).mul_(1.5)
            s["k"], s["v"] = rnd(sum(s["k_len"]), hk, dim), rnd(sum(s["k_len"]), hk, dim)
            s["offsets"] = offsets
            s["k_offsets"] = torch.tensor(_starts(s["k_len"]), dtype=torch.int32, device="cuda")
        if case["mode"] == "train":
            s["do"] = rnd(tokens, hq, dim)
            for n in ("q", "k", "v"):
                s[n] = s[n].detach().requires_grad_()
        return s
    # a cache whose pages lie in any order; the table's unused places hold -1
    each, pages = _pages(case)
    s["k_cache"], s["v_cache"] = rnd(pages, case["page"], hk, dim), rnd(pages, case["page"], hk, dim)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    s["table_rows"] = [order[a:b] for a, b in zip(_starts(each), _starts(each)[1:])]
    wide = max(each)
    s["page_table"] = torch.tensor([r + [-1] * (wide - len(r)) for r in s["table_rows"]], dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(s["k_len"], dtype=torch.int32, device="cuda")
    if case["op"] == "paged":
        new, b = case["new"], case["sequences"]
        s["q"] = (rnd(b, hq, dim) if new == 1 else rnd(b, new, hq, dim)).mul_(1.5)
        return s
    qkv = rnd(tokens, hq + 2 * hk, dim)
    s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
    s["freqs"] = (BASE ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).cuda()
    s["offsets"] = offsets if case["longest"] > 1 else None
    # the plain form's place of each new token: its position, and its row of the cache
    pos, row = [], []
    for n, k, table in zip(s["q_len"], s["k_len"], s["table_rows"]):
        for p in range(k - n, k):
            pos.append(p)
            row.append(table[p // case["page"]] * case["page"] + p % case["page"])
    s["pos"], s["row"] = torch.tensor(pos, device="cuda"), torch.tensor(row, device="cuda")
    return s


# -------------------------------------------------------------------- one pass
def run(s):
    return (_OWN if own else _PLAIN)[s["op"]](s)


def _own_packed(s):
    from prism_b200 import packed_attention
    o = packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["k_offsets"], causal=s["causal"])
    if s["mode"] == "fwd":
        return {"o": o}
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o, "dq": dq, "dk": dk, "dv": dv}


def _own_append(s):
    from prism_b200 import append_paged
    q = append_paged(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"], s["offsets"],
                     q=s["q"], freqs=s["freqs"], layout=s["layout"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_paged(s):
    from prism_b200 import paged_attention
    return {"o": paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])}


def _probabilities(q, k, causal):
    """softmax(q k^T / sqrt(dim)) of [heads, rows, dim] and [heads, keys, dim], 32 bits; with
    `causal` the last row is at the last key, and a row sees the keys up to its own place."""
    rows, keys = q.shape[1], k.shape[1]
    s = (q @ k.transpose(1, 2)).mul_(q.shape[2] ** -0.5)
    if causal:
        at = torch.arange(rows, device=q.device)[:, None] + (keys - rows)
        s.masked_fill_(torch.arange(keys, device=q.device) > at, -math.inf)
    s.sub_(s.amax(2, keepdim=True)).exp_()
    return s.div_(s.sum(2, keepdim=True))


def _plain_packed(s):
    with torch.no_grad():
        group, dim, train = s["hq"] // s["hk"], s["dim"], s["mode"] == "train"
        out = {"o": torch.empty_like(s["q"], memory_format=torch.contiguous_format)}
        if train:
            out |= {"d" + n: torch.zeros(s[n].shape, dtype=torch.float32, device="cuda") for n in ("q", "k", "v")}
        q0, k0 = _starts(s["q_len"]), _starts(s["k_len"])
        for b in range(len(s["q_len"])):
            rows, keys = slice(q0[b], q0[b + 1]), slice(k0[b], k0[b + 1])
            some = max(1, SCORES // (s["q_len"][b] * s["k_len"][b]))    # query heads at a time
            for h in range(0, s["hq"], some):
                h1 = min(s["hq"], h + some)
                of = torch.arange(h, h1, device="cuda") // group        # their key heads
                q = s["q"][rows, h:h1].float().transpose(0, 1)
                k, v = (s[n][keys].index_select(1, of).float().transpose(0, 1) for n in ("k", "v"))
                p = _probabilities(q, k, s["causal"])
                o = p @ v
                out["o"][rows, h:h1] = o.transpose(0, 1).to(s["q"].dtype)
                if not train:
                    continue
                do = s["do"][rows, h:h1].float().transpose(0, 1)
                out["dv"][keys].index_add_(1, of, (p.transpose(1, 2) @ do).transpose(0, 1))
                ds = (do @ v.transpose(1, 2)).sub_((do * o).sum(2, keepdim=True)).mul_(p).mul_(dim ** -0.5)
                out["dq"][rows, h:h1] = (ds @ k).transpose(0, 1)
                out["dk"][keys].index_add_(1, of, (ds.transpose(1, 2) @ q).transpose(0, 1))
        return {n: t.to(s["q"].dtype) for n, t in out.items()}


def _plain_append(s):
    with torch.no_grad():
        angle = s["pos"].double()[:, None] * s["freqs"]     # in 64 bits: far positions
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        rot = s["rot"]

        def turn(x):
            x = x.float()
            if s["layout"] == "interleaved":
                a, b = x[..., 0:rot:2], x[..., 1:rot:2]
                y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
            else:
                a, b = x[..., :rot // 2], x[..., rot // 2:rot]
                y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
            return torch.cat((y, x[..., rot:]), -1).to(s["q"].dtype)

        s["k_cache"].view(-1, s["hk"], s["dim"])[s["row"]] = turn(s["k"])
        s["v_cache"].view(-1, s["hk"], s["dim"])[s["row"]] = s["v"]
        return {"q": turn(s["q"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_paged(s):
    with torch.no_grad():
        b, new, hq, hk, dim = s["sequences"], s["new"], s["hq"], s["hk"], s["dim"]
        q = s["q"].view(b, new, hk, hq // hk, dim).float()
        out = torch.empty_like(q)
        for i, n in enumerate(s["k_len"]):
            pages = s["page_table"][i, :-(-n // s["page"])].long()
            # [hk, keys, dim]
            k, v = (s[c][pages].flatten(0, 1)[:n].float().transpose(0, 1) for c in ("k_cache", "v_cache"))
            sc = torch.einsum("nhgd,hkd->hgnk", q[i], k).mul_(dim ** -0.5)
            if new > 1:
                at = torch.arange(new, device="cuda")[:, None] + (n - new)
                sc.masked_fill_(torch.arange(n, device="cuda") > at, -math.inf)
            p = sc.sub_(sc.amax(3, keepdim=True)).exp_()
            out[i] = torch.einsum("hgnk,hkd->nhgd", p.div_(p.sum(3, keepdim=True)), v)
        return {"o": out.view(s["q"].shape).to(s["q"].dtype)}


_OWN = {"packed": _own_packed, "append": _own_append, "paged": _own_paged}
_PLAIN = {"packed": _plain_packed, "append": _plain_append, "paged": _plain_paged}


# ------------------------------------------------------------------------- work
def work(case):
    q_len, k_len = _lengths(case)
    hq, hk, dim, tokens = case["hq"], case["hk"], case["dim"], sum(q_len)
    if case["op"] == "append":
        # k and v into the cache, q turned, the turned columns' products
        n = tokens * (hq + 2 * hk) * dim
        return {"bytes": 4 * n + 4 * case["rot"] + 4 * tokens, "flops": 3 * tokens * (hq + hk) * case["rot"]}
    causal = case["op"] == "paged" or case["causal"]
    # scores that a row's mask leaves: of n rows at the end of m keys, m - n + 1 .. m
    pairs = sum(n * m - (n * (n - 1) // 2 if causal else 0) for n, m in zip(q_len, k_len))
    q, kv = 2 * tokens * hq * dim, 4 * sum(k_len) * hk * dim
    if case["op"] == "packed" and case["mode"] == "train":
        # q, do in, o and dq out; k, v in, dk, dv out; two products forward, five backward
        return {"bytes": 4 * q + 2 * kv, "flops": 14 * pairs * hq * dim}
    extra = 4 * sum(_pages(case)[0]) if case["op"] == "paged" else 0
    return {"bytes": 2 * q + kv + extra, "flops": 4 * pairs * hq * dim}


# -------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        with torch.no_grad():
            return _exact_append(s)
    if case["op"] == "packed":
        return _exact_packed(s)
    with torch.no_grad():
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda").view(s["sequences"], s["new"], s["hq"], -1)
        group = s["hq"] // s["hk"]
        for i, n in enumerate(s["k_len"]):
            at = torch.arange(n, device="cuda")
            page = torch.tensor(s["table_rows"][i], device="cuda")[at // s["page"]]
            for h in range(s["hq"]):
                k, v = (s[c][page, at % s["page"], h // group].double() for c in ("k_cache", "v_cache"))
                rows = s["q"].view(out.shape)[i, :, h].double()
                out[i, :, h] = _exact_head(rows, k, v, True)
        return {"o": out.view(s["q"].shape)}


def _exact_head(q, k, v, causal):
    score = torch.mm(q, k.t()) / math.sqrt(q.shape[1])
    if causal:
        n, m = score.shape
        score = score.masked_fill(torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1), -math.inf)
    return torch.mm(torch.softmax(score, 1), v)


def _exact_packed(s):
    names = ("q", "k", "v")
    out = {"o": torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")}
    if s["mode"] == "train":
        out |= {"d" + n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in names}
    group, q_at, k_at = s["hq"] // s["hk"], 0, 0
    for n, m in zip(s["q_len"], s["k_len"]):
        for h in range(s["hq"]):
            where = {"q": (slice(q_at, q_at + n), h), "k": (slice(k_at, k_at + m), h // group)}
            where["v"] = where["k"]
            leaf = {t: s[t].detach()[where[t]].double().requires_grad_(s["mode"] == "train") for t in names}
            o = _exact_head(leaf["q"], leaf["k"], leaf["v"], s["causal"])
            out["o"][where["q"]] = o.detach()
            if s["mode"] == "train":
                grads = torch.autograd.grad(o, [leaf[t] for t in names], s["do"][where["q"]].double())
                for t, d in zip(names, grads):
                    out["d" + t][where[t]] += d
        q_at, k_at = q_at + n, k_at + m
    return out


def _exact_append(s):
    out = {n: s[n].double() for n in ("k_cache", "v_cache")}
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda").expand(len(s["pos"]), s["rot"] // 2),
                       s["pos"].double()[:, None] * s["freqs"])[:, None]

    def rotated(x):
        x = x.double()
        half = s["rot"] // 2
        pair = (x[..., :s["rot"]].unflatten(-1, (half, 2)) if s["layout"] == "interleaved"
                else x[..., :s["rot"]].unflatten(-1, (2, half)).transpose(-1, -2))
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        y = y if s["layout"] == "interleaved" else y.transpose(-1, -2)
        return torch.cat((y.flatten(-2), x[..., s["rot"]:]), -1)

    page, place = s["row"] // s["page"], s["row"] % s["page"]
    out["k_cache"][page, place] = rotated(s["k"])
    out["v_cache"][page, place] = s["v"].double()
    return {"q": rotated(s["q"]), "k_cache": out["k_cache"], "v_cache": out["v_cache"]}
