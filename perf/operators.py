"""Measured cases of the operators that answer from retrieved passages.

A search returns passages; a language model reads them as one long prompt that many questions share.  The
operators between the two are measured here, each in its plain form (elementary torch operations in 32 bits) and
as the library's own call:

  page_tables              page tables, cache slots and positions of a batch, from the requests' lengths
  norm_rotate              norm of each head's query and key, position rotation, write into the paged cache
  prompt_attention         attention over packed prompts of different lengths, grouped heads
  shared_prefix_attention  one new token a request, over a prefix that all requests share and over its own pages
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # --- page tables ---------------------------------------------------------------------------------
        # one step of answering: each of 64 requests gets one token, now and then a new page
        dict(name="tables_step_64", op="tables", requests=64, old_lo=1, old_hi=4000, new_lo=1, new_hi=1, page=16,
             base=1000, spare=0, ragged=1),
        # many prompts admitted at once, of 1 to 4,000 tokens each, some of them continued; padded to a fixed total
        dict(name="tables_prompts_1500", op="tables", requests=1500, old_lo=0, old_hi=700, new_lo=1, new_hi=4000,
             page=32, base=0, spare=777, ragged=2),
        # --- norm, rotation and cache write ----------------------------------------------------------------
        # one token of each of 33 requests; the keys go to the cache only
        dict(name="rotate_step_33", op="rotate", type="bf16", tokens=33, heads=32, kv_heads=8, dim=128, turned=128,
             pairs=False, page=16, keep_k=False, longest=40000, skipped=0),
        # a prompt of odd length, half of each head rotated in neighbouring pairs, a few padding tokens
        dict(name="rotate_prompt_1777_pairs", op="rotate", type="f16", tokens=1777, heads=12, kv_heads=12, dim=64,
             turned=32, pairs=True, page=64, keep_k=True, longest=4096, skipped=9),
        # the prompts of a large batch
        dict(name="rotate_prompt_50000", op="rotate", type="bf16", tokens=50000, heads=32, kv_heads=8, dim=128,
             turned=128, pairs=False, page=32, keep_k=True, longest=131072, skipped=100),
        # --- attention over prompts ------------------------------------------------------------------------
        # the smallest call: three short questions, one of a single token
        dict(name="prompt_3_questions", op="prompt", type="bf16", requests=3, lo=1, hi=60, history=0, heads=32,
             kv_heads=8, dim=128, causal=True, stats=False, ragged=3),
        # passages embedded by an encoder (each token sees its whole passage), twelve heads of 64
        dict(name="prompt_passages_200", op="prompt", type="f16", requests=200, lo=16, hi=500, history=0, heads=12,
             kv_heads=12, dim=64, causal=False, stats=False, ragged=4),
        # an ordinary batch of prompts, packed, one to four thousand tokens
        dict(name="prompt_packed_24", op="prompt", type="bf16", requests=24, lo=1, hi=4000, history=0, heads=32,
             kv_heads=8, dim=128, causal=True, stats=False, ragged=5),
        # one long prompt of retrieved passages: the largest
        dict(name="prompt_long_16k", op="prompt", type="bf16", requests=1, lo=16384, hi=16384, history=0, heads=32,
             kv_heads=8, dim=128, causal=True, stats=True, ragged=6),
        # --- attention with a shared prefix ----------------------------------------------------------------
        # a handful of questions over one short passage
        dict(name="shared_4_over_700", op="shared", type="bf16", requests=4, prefix=700, lo=0, hi=40, heads=32,
             kv_heads=8, dim=128, page=16, stats=False, ragged=7),
        # an ordinary batch, seven query heads to a key head
        dict(name="shared_61_over_8000", op="shared", type="f16", requests=61, prefix=8000, lo=1, hi=600, heads=28,
             kv_heads=4, dim=128, page=32, stats=True, ragged=8),
        # a large batch over long retrieved context, answers of up to 1,500 tokens
        dict(name="shared_256_over_20000", op="shared", type="bf16", requests=256, prefix=20001, lo=1, hi=1500,
             heads=32, kv_heads=8, dim=128, page=64, stats=False, ragged=9),
    ]


# Head layouts (query heads, key heads, head size) that cases are drawn from.
_HEADS = [(32, 8, 128), (8, 2, 128), (16, 2, 128), (28, 4, 128), (12, 12, 128), (8, 1, 128), (16, 4, 64), (12, 12, 64),
          (32, 4, 64), (20, 4, 96), (10, 5, 80)]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    return n - 1 if n == 3072 else n


def _drawn(rng):
    op = rng.choice(["tables", "rotate", "prompt", "shared"])
    c = {"op": op, "ragged": rng.randrange(1 << 30)}
    if op == "tables":
        hi = _log(rng, 1, 4000)
        return c | {"requests": _log(rng, 1, 1500), "old_lo": 0, "old_hi": _log(rng, 1, 4000),
                    "new_lo": rng.choice([0, 1, hi]), "new_hi": hi, "page": rng.choice([16, 32, 64, 128]),
                    "base": rng.choice([0, _log(rng, 1, 30000)]), "spare": rng.choice([0, _log(rng, 1, 999)])}
    heads, kv, dim = rng.choice(_HEADS)
    c |= {"type": rng.choice(["bf16", "bf16", "f16"]), "heads": heads, "kv_heads": kv, "dim": dim}
    if op == "rotate":
        tokens = _log(rng, 1, 50000)
        c.pop("ragged")
        return c | {"tokens": tokens, "turned": rng.choice([dim, dim, 32]), "pairs": rng.random() < 0.3,
                    "page": rng.choice([16, 32, 64, 128]), "keep_k": rng.random() < 0.5,
                    "longest": _log(rng, 2048, 131072), "skipped": rng.randrange(min(tokens, 50))}
    if op == "prompt":
        hi = _log(rng, 1, 16384)
        return c | {"requests": _log(rng, 1, 200), "lo": rng.choice([0, 1, max(1, hi // 2), hi]), "hi": hi,
                    "history": rng.choice([0, 0, _log(rng, 1, 16384)]), "causal": rng.random() < 0.75,
                    "stats": rng.random() < 0.3}
    return c | {"requests": _log(rng, 1, 256), "prefix": rng.choice([0, _log(rng, 16, 20000), _log(rng, 300, 20000)]),
                "lo": rng.choice([0, 1]), "hi": _log(rng, 1, 1500), "page": rng.choice([16, 32, 64, 128]),
                "stats": rng.random() < 0.3}


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        c = _drawn(rng)
        w, m = work(c), most[c["op"]]
        # the plain form pads each request to the longest: what that makes of the batch stays within bounds too
        if c["op"] == "prompt":
            padded = c["requests"] * c["hi"] * (c["hi"] + c["history"]) * c["heads"]
            if padded > 32 * 16384 ** 2 or c["requests"] * (c["hi"] + c["history"]) * c["heads"] * c["dim"] > 1 << 30:
                continue
        if w["flops"] <= m["flops"] and w["bytes"] <= m["bytes"]:
            return c


def _lengths(case, lo, hi, salt=0):
    """Lengths of the case's requests: spread over the logarithm, the longest among them."""
    rng = random.Random(case["ragged"] * 16 + salt)
    n = [int(round(math.exp(rng.uniform(math.log(max(lo, 0) + 0.5), math.log(hi + 0.5))) - 0.01)) for _ in
         range(case["requests"])]
    n = [max(lo, min(hi, x)) for x in n]
    n[rng.randrange(len(n))] = hi
    return n


def _prompt_lengths(case):
    new = _lengths(case, case["lo"], case["hi"])
    old = _lengths(case, 0, case["history"], 1) if case["history"] else [0] * len(new)
    return new, [a + b for a, b in zip(new, old)]


def _pages(n, page):
    return -(-n // page)


def work(case):
    op = case["op"]
    if op == "tables":
        old, new = _lengths(case, case["old_lo"], case["old_hi"]), _lengths(case, case["new_lo"], case["new_hi"], 1)
        page = case["page"]
        more = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(old, new))
        tokens = sum(new) + case["spare"]
        # lengths and free pages in; table entries, lengths, starts, positions and slots out
        return {"bytes": 8 * len(old) + 8 * more + 8 * len(old) + 12 * tokens, "flops": 0}
    width = case["heads"] + 2 * case["kv_heads"]
    if op == "rotate":
        t, d = case["tokens"], case["dim"]
        out = case["heads"] + (2 + (1 if case["keep_k"] else 0)) * case["kv_heads"]
        return {"bytes": 2 * t * d * (width + out) + 4 * t * case["turned"] + 12 * t,
                "flops": t * (case["heads"] + case["kv_heads"]) * (4 * d + 3 * case["turned"])}
    d, heads, kv = case["dim"], case["heads"], case["kv_heads"]
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        pairs = sum(a * b - (a * (a - 1) // 2 if case["causal"] else 0) for a, b in zip(lq, lk))
        return {"bytes": 2 * d * (2 * heads * sum(lq) + 2 * kv * sum(lk)) + (4 * heads * sum(lq) if case["stats"] else 0),
                "flops": 4 * d * heads * pairs}
    n, p = _lengths(case, case["lo"], case["hi"]), case["prefix"]
    b = len(n)
    return {"bytes": 2 * d * (2 * heads * b + 2 * kv * (sum(n) + p)) + (4 * heads * b if case["stats"] else 0)
            + 4 * sum(_pages(x, case["page"]) for x in n) + 4 * b,
            "flops": 4 * d * heads * (sum(n) + b * p)}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    op, s = case["op"], {"case": case}
    if op == "tables":
        old, new = _lengths(case, case["old_lo"], case["old_hi"]), _lengths(case, case["new_lo"], case["new_hi"], 1)
        page = case["page"]
        had, more = [_pages(a, page) for a in old], sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(old, new))
        width = max(_pages(a + b, page) for a, b in zip(old, new)) + 3
        order = torch.randperm(sum(had) + more + 5, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(old), width), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(width, device="cuda")[None] < ints(had)[:, None]
        table[held] = order[:sum(had)]
        return s | {"old": ints(old), "new": ints(new), "free": order[sum(had):], "table": table,
                    "total": sum(new) + case["spare"]}
    dtype, heads, kv, d = _TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    if op == "rotate":
        t, page, r = case["tokens"], case["page"], case["turned"]
        x = normal(t, heads + 2 * kv, d) * 3  # the projection's output: queries, keys and values of each token
        pages = _pages(t, page) + 2
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
        if case["skipped"]:  # padding tokens at the end
            slots[t - case["skipped"]:] = -1
        turn = torch.arange(case["longest"], device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        return s | {"q": x[:, :heads], "k": x[:, heads:heads + kv], "v": x[:, heads + kv:], "slots": slots,
                    "positions": torch.randint(0, case["longest"], (t,), generator=g, device="cuda", dtype=torch.int32),
                    "turns": torch.cat([turn.cos(), turn.sin()], 1).float(),
                    "q_weight": 1 + normal(d) / 4, "k_weight": 1 + normal(d) / 4,
                    "k_cache": torch.zeros(pages, page, kv, d, dtype=dtype, device="cuda"),
                    "v_cache": torch.zeros(pages, page, kv, d, dtype=dtype, device="cuda")}
    if op == "prompt":
        lq, lk = _prompt_lengths(case)
        fused = normal(sum(lk), 2 * kv, d)  # values are a slice of the projection's output
        start = lambda n: ints([0] + n).cumsum(0).to(torch.int32)  # noqa: E731
        return s | {"q": normal(sum(lq), heads, d) * 2, "k": normal(sum(lk), kv, d), "v": fused[:, kv:],
                    "starts": start(lq), "starts_k": start(lk) if case["history"] else None,
                    "longest": max(lq), "longest_k": max(lk)}
    n, p, page = _lengths(case, case["lo"], case["hi"]), case["prefix"], case["page"]
    shared, width = _pages(p, page), max(1, max(_pages(x, page) for x in n))
    total = shared + sum(_pages(x, page) for x in n)
    order = torch.randperm(total + 1, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(n), width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None] < ints([_pages(x, page) for x in n])[:, None]
    table[held] = order[shared:total]
    return s | {"q": normal(len(n), heads, d) * 2, "k_cache": normal(total + 1, page, kv, d),
                "v_cache": normal(total + 1, page, kv, d), "prefix_pages": order[:shared], "table": table,
                "lengths": ints(n)}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if own:
        import vesper_db_b200 as vesper
        if c["op"] == "tables":
            return list(vesper.page_tables(s["old"], s["new"], s["free"], s["table"], c["page"], s["total"],
                                           base=c["base"]))
        if c["op"] == "rotate":
            q, k = vesper.norm_rotate(s["q"], s["k"], s["v"], s["positions"], s["turns"], q_weight=s["q_weight"],
                                      k_weight=s["k_weight"], eps=1e-6, pairs=c["pairs"], slots=s["slots"],
                                      k_cache=s["k_cache"], v_cache=s["v_cache"], keep_k=c["keep_k"])
            return [q, k, s["k_cache"], s["v_cache"]]
        if c["op"] == "prompt":
            return vesper.prompt_attention(s["q"], s["k"], s["v"], s["starts"], s["starts_k"], causal=c["causal"],
                                           stats=c["stats"])
        return vesper.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], c["prefix"],
                                              s["table"], s["lengths"], stats=c["stats"])
    return {"tables": _tables, "rotate": _rotate, "prompt": _prompt, "shared": _shared}[c["op"]](s)


def _tables(s):
    c, old, new, table, page = s["case"], s["old"], s["new"], s["table"], s["case"]["page"]
    after = old + new
    had, need = (old + (page - 1)) // page, (after + (page - 1)) // page
    ends = torch.cumsum(new, 0)
    first = torch.cumsum(need - had, 0) - (need - had)
    at = torch.arange(table.shape[1], device=table.device)[None]
    taken = first[:, None] + at - had[:, None]
    fresh = (at >= had[:, None]) & (at < need[:, None])
    table.copy_(torch.where(fresh, s["free"][taken.clamp(0, s["free"].shape[0] - 1)], table))
    token = torch.arange(s["total"], device=table.device)
    row = torch.searchsorted(ends, token.to(ends.dtype), right=True)
    real = row < old.shape[0]
    row = torch.where(real, row, 0)
    where = old[row] + token - (ends[row] - new[row])
    where = torch.where(real, where, 0)
    slot = table[row, where // page].long() * page + where % page
    starts = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
    return [table, after, starts, torch.where(real, where + c["base"], 0).to(torch.int32), torch.where(real, slot, -1),
            (need - had).sum(dtype=torch.int32).reshape(1)]


def _turned(x, weight, turns, pairs):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    r = turns.shape[-1]
    cos, sin = turns[:, None, :r // 2], turns[:, None, r // 2:]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if pairs else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _rotate(s):
    c, dtype = s["case"], s["q"].dtype
    turns = s["turns"][s["positions"].long()]
    q = _turned(s["q"], s["q_weight"], turns, c["pairs"]).to(dtype)
    k = _turned(s["k"], s["k_weight"], turns, c["pairs"]).to(dtype)
    kept = s["slots"] >= 0
    rows = s["slots"][kept]
    s["k_cache"].flatten(0, 1)[rows] = k[kept]
    s["v_cache"].flatten(0, 1)[rows] = s["v"][kept]
    return [q, k if c["keep_k"] else None, s["k_cache"], s["v_cache"]]


def _padded(x, starts, longest):
    """[requests, longest, heads, size] in 32 bits of a packed [tokens, heads, size], and which rows are real."""
    at = torch.arange(longest, device=x.device)[None]
    real = at < (starts[1:] - starts[:-1])[:, None]
    return x[torch.where(real, starts[:-1, None] + at, 0).long()].float(), real


def _prompt(s):
    c = s["case"]
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    starts, starts_k = s["starts"], s["starts"] if s["starts_k"] is None else s["starts_k"]
    q, real = _padded(s["q"], starts, s["longest"])
    k, real_k = _padded(s["k"], starts_k, s["longest_k"])
    v, _ = _padded(s["v"], starts_k, s["longest_k"])
    v = torch.where(real_k[..., None, None], v, 0.0)
    b, group = q.shape[0], heads // kv
    q = q.view(b, -1, kv, group, d).permute(0, 2, 3, 1, 4)
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    seen = real_k[:, None, None, None, :]
    if c["causal"]:  # the last token sees every key, each one before it sees one key less
        lq, lk = starts[1:] - starts[:-1], starts_k[1:] - starts_k[:-1]
        last = torch.arange(s["longest"], device=q.device)[None] + (lk - lq)[:, None]
        seen = seen & (torch.arange(s["longest_k"], device=q.device) <= last[:, None, None, :, None])
    out = torch.empty(b, kv, group, s["longest"], d, device=q.device)
    lse = torch.empty(b, kv, group, s["longest"], device=q.device)
    step = max(1, (1 << 30) // (b * group * s["longest"] * s["longest_k"]))
    for h in range(0, kv, step):  # as many heads at once as 4 GiB of scores hold
        score = q[:, h:h + step] @ k[:, h:h + step, None] / math.sqrt(d)
        score = score.masked_fill_(~seen, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
        score = score.sub_(top).exp_()
        total = score.sum(-1, keepdim=True)
        out[:, h:h + step] = score @ v[:, h:h + step, None] / torch.where(total > 0, total, 1.0)
        lse[:, h:h + step] = (top + total.log())[..., 0]
        del score
    out = out.permute(0, 3, 1, 2, 4).reshape(b, -1, heads, d)
    at = torch.arange(s["q"].shape[0], device=q.device)
    row = torch.searchsorted(starts[1:].contiguous(), at.to(starts.dtype), right=True)
    col = at - starts[row]
    out = out[row, col].to(s["q"].dtype)
    return [out, lse.permute(0, 3, 1, 2).reshape(b, -1, heads)[row, col]] if c["stats"] else out


def _shared(s):
    c, q, kc, vc = s["case"], s["q"], s["k_cache"], s["v_cache"]
    heads, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    b, group = q.shape[0], heads // kv
    q = q.float().view(b, kv, group, d)
    width = s["table"].shape[1] * page
    own_at = s["table"].long().clamp(min=0)
    at = torch.arange(width, device=q.device)[None]
    k = kc[own_at].view(b, width, kv, d).float()
    v = vc[own_at].view(b, width, kv, d).float()
    seen = at < s["lengths"][:, None]
    v = torch.where(seen[..., None, None], v, 0.0)
    mine = torch.einsum("bkgd,bnkd->bkgn", q, k) / math.sqrt(d)
    mine = mine.masked_fill(~seen[:, None, None], -math.inf)
    pk = kc[s["prefix_pages"].long()].flatten(0, 1)[:c["prefix"]].float()
    pv = vc[s["prefix_pages"].long()].flatten(0, 1)[:c["prefix"]].float()
    theirs = torch.einsum("bkgd,nkd->bkgn", q, pk) / math.sqrt(d)
    top = torch.cat([mine, theirs], -1).amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    mine, theirs = (mine - top).exp(), (theirs - top).exp()
    total = mine.sum(-1, keepdim=True) + theirs.sum(-1, keepdim=True)
    out = torch.einsum("bkgn,bnkd->bkgd", mine, v) + torch.einsum("bkgn,nkd->bkgd", theirs, pv)
    out = (out / torch.where(total > 0, total, 1.0)).reshape(b, heads, d).to(s["q"].dtype)
    return [out, (top + total.log())[..., 0].reshape(b, heads)] if c["stats"] else out


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What run() returns, from the definitions, one request (and one block of queries) at a time, in 64 bits."""
    s, op = prepare(case, seed), case["op"]
    if op == "tables":
        return None
    if op == "rotate":
        return _exact_rotate(s, case)
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    if op == "prompt":
        starts = s["starts"].tolist()
        starts_k = starts if s["starts_k"] is None else s["starts_k"].tolist()
        for i in range(len(starts) - 1):
            k, v = (s[x][starts_k[i]:starts_k[i + 1]].double().transpose(0, 1) for x in ("k", "v"))
            lq, lk = starts[i + 1] - starts[i], k.shape[1]
            if lk == 0:
                continue
            for a in range(0, lq, 2048):
                e = min(a + 2048, lq)
                rows = slice(starts[i] + a, starts[i] + e)
                for h in range(heads):
                    x = s["q"][rows, h].double() @ k[h // group].T * d ** -0.5
                    if case["causal"]:
                        x = x + torch.full_like(x, -math.inf).triu(a + lk - lq + 1)
                    empty = torch.isneginf(x).all(1)
                    lse[rows, h] = torch.logsumexp(x, 1)
                    out[rows, h] = torch.where(empty[:, None], 0.0, torch.softmax(x, 1) @ v[h // group])
    else:
        n, p = s["lengths"].tolist(), case["prefix"]
        pk, pv = (s[x][s["prefix_pages"].long()].double().reshape(-1, kv, d)[:p] for x in ("k_cache", "v_cache"))
        for i, m in enumerate(n):
            held = s["table"][i, :_pages(m, case["page"])].long()
            k, v = (torch.cat([shared, s[x][held].double().reshape(-1, kv, d)[:m]]).transpose(0, 1)
                    for shared, x in ((pk, "k_cache"), (pv, "v_cache")))
            if k.shape[1] == 0:
                continue
            x = s["q"][i].double().view(kv, group, d) @ k.transpose(1, 2) * d ** -0.5
            lse[i] = torch.logsumexp(x, -1).reshape(-1)
            out[i] = (torch.softmax(x, -1) @ v).reshape(heads, d)
    return [out, lse] if case["stats"] else out


def _exact_rotate(s, case):
    r = case["turned"]
    i = torch.arange(r, device="cuda")
    mate = (i ^ 1) if case["pairs"] else (i + r // 2) % r
    angle = (i // 2) if case["pairs"] else i % (r // 2)
    sign = torch.where((i % 2 == 0) if case["pairs"] else (i < r // 2), -1.0, 1.0).double()
    turns = s["turns"][s["positions"].long()].double()

    def turned(x, w):
        x = x.double()
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        cos, sin = turns[:, None, angle], turns[:, None, r // 2 + angle]
        x[..., :r] = x[..., :r] * cos + sign * x[..., mate] * sin
        return x

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    kept = s["slots"] >= 0
    k_cache.view(-1, *k_cache.shape[2:])[s["slots"][kept]] = k[kept]
    v_cache.view(-1, *v_cache.shape[2:])[s["slots"][kept]] = s["v"][kept].double()
    return [q, k if case["keep_k"] else None, k_cache, v_cache]
