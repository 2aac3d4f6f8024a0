"""The operators of chunked prompts and drafted tokens, and the cases they are measured on.

A server that continues a prompt in chunks, or that checks several drafted tokens of each request in one pass, appends
chunks of new tokens to the paged cache ("append"), attends from each chunk over everything its sequence has cached
("attention"), turns the logits of every row into probabilities ("probs") and accepts or replaces the drafts
("verify"). `run` has each of them in a plain form of elementary torch operations, and as the calls of vortex_b200.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one speculative step of a batch of 32: up to five new tokens each, the decoder's 32 heads of 128
        dict(name="append drafts", op="append", seqs=32, new_lo=1, new_hi=5, past_lo=1000, past_hi=2100, heads=32, dim=128, block=16),
        # prompts that arrive together, some continuing a shared prefix
        dict(name="append prompts", op="append", seqs=6, new_lo=1001, new_hi=4096, past_lo=1, past_hi=777, heads=8, dim=128, block=16),
        # a single user: four drafts on a short conversation, where latency counts
        dict(name="one user's drafts", op="attention", seqs=1, new_lo=4, new_hi=4, ctx_lo=333, ctx_hi=333, q_heads=32, kv_heads=32, dim=128, block=16, kv="bf16"),
        # the decoder's own shape at batch 32: every request checks one to five tokens
        dict(name="drafts of 32 requests", op="attention", seqs=32, new_lo=1, new_hi=5, ctx_lo=1024, ctx_hi=2101, q_heads=32, kv_heads=32, dim=128, block=16, kv="bf16"),
        # grouped heads over an int8 cache, longer contexts, longer drafts
        dict(name="drafts, grouped, int8", op="attention", seqs=32, new_lo=4, new_hi=8, ctx_lo=1025, ctx_hi=8192, q_heads=32, kv_heads=8, dim=128, block=16, kv="int8"),
        # few sequences over very long contexts, heads of 64
        dict(name="long contexts, d 64", op="attention", seqs=3, new_lo=1, new_hi=16, ctx_lo=20001, ctx_hi=32768, q_heads=16, kv_heads=4, dim=64, block=32, kv="bf16"),
        # a mixed batch: short prompts' chunks of ragged lengths, int8 cache
        dict(name="ragged chunks, int8", op="attention", seqs=5, new_lo=61, new_hi=700, ctx_lo=700, ctx_hi=2048, q_heads=32, kv_heads=32, dim=128, block=16, kv="int8"),
        # a chunk of a long prompt
        dict(name="chunk of a long prompt", op="attention", seqs=1, new_lo=4096, new_hi=4096, ctx_lo=16384, ctx_hi=16384, q_heads=32, kv_heads=8, dim=128, block=16, kv="bf16"),
        # five rows of one request (four drafts and the row behind them)
        dict(name="probs of one request", op="probs", rows=5, vocab=32000, temperature=0.8, banned=0),
        # a batch's rows over a large vocabulary of odd size, with tokens that a grammar bans
        dict(name="probs of a batch", op="probs", rows=160, vocab=131071, temperature=1.0, banned=1000),
        # one request, four drafts of a draft model
        dict(name="verify one request", op="verify", requests=1, drafts_lo=4, drafts_hi=4, vocab=32000, draft_probs=True),
        # a batch with up to eight drafts each over a large vocabulary
        dict(name="verify a batch", op="verify", requests=64, drafts_lo=1, drafts_hi=8, vocab=131072, draft_probs=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "probs", "verify"])
    if op == "append":
        seqs = _log(rng, 1, 48)
        new_hi = _log(rng, 1, max(1, 20000 // seqs))
        past_hi = rng.randint(3, 2100)
        heads, dim = rng.choice([1, 2, 4, 8, 32]), rng.choice([64, 128])
        return dict(op=op, seqs=seqs, new_lo=max(1, new_hi // rng.randint(1, 5)), new_hi=new_hi, past_lo=past_hi // 3, past_hi=past_hi, heads=heads, dim=dim,
                    block=rng.choice([16, 16, 32, 64]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
        group = rng.choice([1, 2, 3, 4, 6, 8]) if kv_heads < 32 else 1
        dim, kind, block = rng.choice([64, 128]), rng.choice(["bf16", "bf16", "int8"]), rng.choice([16, 16, 32, 64])
        if rng.random() < 0.55:  # drafts
            seqs, new_hi, ctx_hi = _log(rng, 1, 40), rng.randint(1, 16), _log(rng, 17, 8192)
        else:  # chunks of prompts
            seqs, new_hi = _log(rng, 1, 6), _log(rng, 17, 2000)
            ctx_hi = new_hi + _log(rng, 1, 6000)
        while seqs > 1 and seqs * ctx_hi * kv_heads * dim > 40e6:  # what the plain form can hold
            seqs = max(1, seqs // 2)
        while ctx_hi > 17 and seqs * new_hi * ctx_hi * kv_heads * group > 1.0e9:
            new_hi, ctx_hi = max(1, new_hi * 3 // 4), max(17, ctx_hi * 3 // 4)
        ctx_hi = max(ctx_hi, new_hi)
        return dict(op=op, seqs=seqs, new_lo=max(1, new_hi // rng.randint(1, 4)), new_hi=new_hi, ctx_lo=max(new_hi, ctx_hi // rng.randint(1, 3)), ctx_hi=ctx_hi,
                    q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, block=block, kv=kind)
    vocab = _log(rng, 500, 131072)
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, max(1, min(400, 20_000_000 // vocab))), vocab=vocab, temperature=rng.choice([0.3, 0.7, 1.0, 1.5]), banned=rng.choice([0, vocab // 10]))
    drafts_hi = rng.randint(1, 8)
    return dict(op=op, requests=_log(rng, 1, max(1, min(64, 60_000_000 // (vocab * (drafts_hi + 1))))), drafts_lo=rng.randint(0, drafts_hi), drafts_hi=drafts_hi, vocab=vocab,
                draft_probs=rng.random() < 0.7)


def _spread(lo, hi, n):
    """n sizes between lo and hi, both among them, in no order of size."""
    return [lo + (hi - lo) * (i * 7 % n) // max(1, n - 1) for i in range(n)] if n % 7 else [lo + (hi - lo) * (i * 5 % n) // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens cached when the call is made) of each sequence."""
    n = case["seqs"]
    new = _spread(case["new_lo"], case["new_hi"], n)
    if case["op"] == "append":
        return new, _spread(case["past_lo"], case["past_hi"], n)[::-1]
    return new, [max(c, m) for c, m in zip(_spread(case["ctx_lo"], case["ctx_hi"], n)[::-1], new)]


def work(case):
    if case["op"] == "append":
        new, _ = _lengths(case)
        row = 2 * case["heads"] * case["dim"] * 2
        return {"bytes": 2 * sum(new) * row + 4 * sum(-(-m // case["block"]) for m in new), "flops": 0}
    if case["op"] == "attention":
        new, ctx = _lengths(case)
        token = 2 * case["kv_heads"] * (case["dim"] * 2 if case["kv"] == "bf16" else case["dim"] + 4)
        seen = sum(m * c - m * (m - 1) // 2 for m, c in zip(new, ctx))
        return {"bytes": sum(ctx) * token + sum(new) * case["q_heads"] * (4 * case["dim"] + 4), "flops": 4 * seen * case["q_heads"] * case["dim"]}
    if case["op"] == "probs":
        return {"bytes": 8 * case["rows"] * case["vocab"], "flops": 4 * case["rows"] * case["vocab"]}
    drafts = sum(_spread(case["drafts_lo"], case["drafts_hi"], case["requests"]))
    # the probabilities of the drafted tokens, and one row of each model for the token that is drawn
    rows = 2 if case["draft_probs"] else 1
    return {"bytes": 4 * case["requests"] * (case["vocab"] * rows + 3) + 20 * drafts, "flops": 3 * case["requests"] * case["vocab"]}


# ---------------------------------------------------------------- inputs

def _values(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE).to(torch.bfloat16)


def _ints(v):
    return torch.tensor(v, dtype=torch.int64, device=DEVICE)


def _cache(case, tokens, k, v, room):
    """A paged cache that holds tokens[i] tokens of sequence i (k, v: their rows, one sequence after another) and has room[i]
    tokens' blocks for it in all: the framework's own, or plain pages with the blocks handed out in the same order."""
    heads, dim, block, n = k.shape[1], case["dim"], case["block"], len(tokens)
    need = sum(-(-r // block) for r in room) + n
    most = max(-(-r // block) for r in room)
    kind = case.get("kv", "bf16")
    if own:
        from vortex_b200 import kv_cache

        c = kv_cache.PagedKVCache(1, heads, dim, block_size=block, max_blocks=need, max_seqs=n, max_blocks_per_seq=most,
                                  kv_dtype=kv_cache.I8 if kind == "int8" else kv_cache.BF16)
        pages = c.pages()
        if kind == "bf16":
            pages["k"].zero_()
            pages["v"].zero_()
        c.append_chunks(0, np.arange(n, dtype=np.int64), np.asarray(tokens, dtype=np.int32), k, v)
        if kind == "int8":
            # a code whose quotient lies on the border between two falls either way with the last bit of the scale: the
            # cache gets the very codes that the plain form attends over
            for name, made in _plain_cache(case, tokens, k, v, room).items():
                if name in ("k", "v", "k_scale", "v_scale"):
                    pages[name].copy_(made)
        return {"cache": c, **pages}
    tables = torch.full((1, n, most), -1, dtype=torch.int32, device=DEVICE)
    first, at = 0, []
    for i, t in enumerate(tokens):
        blocks = -(-t // block)
        tables[0, i, :blocks] = torch.arange(first, first + blocks, device=DEVICE)
        at.append(torch.arange(t, device=DEVICE) + first * block)
        first += blocks
    slots = torch.cat(at) if at else _ints([])
    made = {"tables": tables, "lens": torch.tensor([tokens], dtype=torch.int32, device=DEVICE), "used": first}
    for name, rows in (("k", k), ("v", v)):
        if kind == "int8":  # one scale for each token and head: the largest magnitude over 127, codes rounded half away from zero
            x = rows.double()
            s = x.abs().amax(-1) / 127.0
            s = torch.where(s == 0, torch.ones_like(s), s)
            c = x / s[..., None]
            codes = (torch.sign(c) * torch.floor(c.abs() + 0.5)).clamp(-128, 127).to(torch.int8)
            pages, scales = torch.zeros(need, heads, block, dim, dtype=torch.int8, device=DEVICE), torch.ones(need, heads, block, device=DEVICE)
            pages[slots // block, :, slots % block] = codes
            scales[slots // block, :, slots % block] = s.float()
            made[name + "_scale"] = scales
        else:
            pages = torch.zeros(need, heads, block, dim, dtype=torch.bfloat16, device=DEVICE)
            pages[slots // block, :, slots % block] = rows
        made[name] = pages
    return made


def _plain_cache(*args):
    """What _cache makes for the plain form, for a framework's cache that has to hold the same."""
    global own
    own = False
    try:
        return _cache(*args)
    finally:
        own = True


def _inputs(case, seed):
    """The values of a case, from the seed alone."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "append":
        new, past = _lengths(case)
        return {name: _values(gen, sum(t), case["heads"], case["dim"]) for name, t in (("k_past", past), ("v_past", past), ("k", new), ("v", new))}
    if case["op"] == "attention":
        new, ctx = _lengths(case)
        x = {name: _values(gen, sum(ctx), case["kv_heads"], case["dim"]) for name in ("k", "v")}
        x["q"] = (2.0 * torch.randn(sum(new), case["q_heads"], case["dim"], generator=gen, device=DEVICE)).to(torch.bfloat16)
        return x
    if case["op"] == "probs":
        logits = 2.5 * torch.randn(case["rows"], case["vocab"], generator=gen, device=DEVICE)
        if case["banned"]:
            logits[:, torch.randperm(case["vocab"], generator=gen, device=DEVICE)[: case["banned"]]] = -math.inf
        return {"logits": logits}
    counts = _spread(case["drafts_lo"], case["drafts_hi"], case["requests"])
    rows, drafts = sum(counts) + case["requests"], sum(counts)
    logits = 3.0 * torch.randn(rows, case["vocab"], generator=gen, device=DEVICE)
    of = torch.repeat_interleave(_ints(range(case["requests"])), _ints(counts))
    behind = torch.arange(drafts, device=DEVICE) + of  # a draft's row of the target: one row more for each request before it
    near = torch.softmax(logits[behind] + 0.7 * torch.randn(drafts, case["vocab"], generator=gen, device=DEVICE), -1)
    tokens = torch.multinomial(near, 1, generator=gen).reshape(-1) if drafts else _ints([])
    return {"target": torch.softmax(logits, -1), "draft": near if case["draft_probs"] else None, "drafts": tokens.to(torch.int32),
            "u_accept": torch.rand(drafts, generator=gen, device=DEVICE), "u_sample": torch.rand(case["requests"], generator=gen, device=DEVICE)}


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case}
    if case["op"] == "append":
        new, past = _lengths(case)
        s |= {"k_new": x["k"], "v_new": x["v"], "ids": np.arange(case["seqs"], dtype=np.int64), "new": np.asarray(new, dtype=np.int32), "past": np.asarray(past, dtype=np.int64),
              "new_d": _ints(new), "past_d": _ints(past)}
        s |= _cache(case, past, x["k_past"], x["v_past"], [a + b for a, b in zip(new, past)])
    elif case["op"] == "attention":
        new, ctx = _lengths(case)
        s |= {"q": x["q"], "ids": np.arange(case["seqs"], dtype=np.int64), "new": np.asarray(new, dtype=np.int32), "new_d": _ints(new), "ctx_d": _ints(ctx), "most": max(new), "longest": max(ctx)}
        s["lse"] = torch.empty(sum(new), case["q_heads"], device=DEVICE)
        s |= _cache(case, ctx, x["k"], x["v"], ctx)
    elif case["op"] == "probs":
        s |= x
    else:
        counts = _spread(case["drafts_lo"], case["drafts_hi"], case["requests"])
        s |= x | {"counts": np.asarray(counts, dtype=np.int32), "counts_d": _ints(counts), "most": max(counts)}
    return s


# ---------------------------------------------------------------- the framework's calls

def _run_own(s):
    op = s["case"]["op"]
    if op == "append":
        c = s["cache"]
        c.truncate(s["ids"], s["past"])  # what an earlier pass appended is taken back, as rejected drafts are
        c.append_chunks(0, s["ids"], s["new"], s["k_new"], s["v_new"])
        return {"k": s["k"], "v": s["v"], "tables": s["tables"], "lens": s["lens"]}
    if op == "attention":
        return {"out": s["cache"].chunk_attention(0, s["ids"], s["new"], s["q"], lse=s["lse"]), "lse": s["lse"]}
    from vortex_b200 import sampling

    if op == "probs":
        return sampling.token_probs(s["logits"], s["case"]["temperature"])
    tokens, accepted = sampling.verify_drafts(s["drafts"], s["counts"], s["target"], s["draft"], s["u_accept"], s["u_sample"])
    return {"tokens": tokens, "accepted": accepted}


# ---------------------------------------------------------------- the plain forms

def _rows_of(counts, total):
    """For each packed row: its sequence, and its place in it."""
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=DEVICE), counts, output_size=total)
    return seq, torch.arange(total, device=DEVICE) - (torch.cumsum(counts, 0) - counts)[seq]


def _plain_append(s):
    block, new, past = s["case"]["block"], s["new_d"], s["past_d"]
    total = s["k_new"].shape[0]
    seq, place = _rows_of(new, total)
    pos = past[seq] + place
    held = (past + block - 1) // block
    more = (past + new + block - 1) // block - held
    first = s["used"] + torch.cumsum(more, 0) - more  # the first new block of each sequence
    index = pos // block
    fresh = index - held[seq]
    tables = s["tables"][0]
    ids = torch.where(fresh >= 0, first[seq] + fresh, tables[seq, index].long())
    tables[seq, index] = ids.to(torch.int32)
    s["k"][ids, :, pos % block] = s["k_new"]
    s["v"][ids, :, pos % block] = s["v_new"]
    s["lens"][0] = (past + new).to(torch.int32)
    return {"k": s["k"], "v": s["v"], "tables": s["tables"], "lens": s["lens"]}


def _plain_attention(s):
    case, new, ctx = s["case"], s["new_d"], s["ctx_d"]
    n, most, longest = case["seqs"], s["most"], s["longest"]
    hk, dim, block = case["kv_heads"], case["dim"], case["block"]
    group = case["q_heads"] // hk
    blocks = -(-longest // block)
    table = s["tables"][0][:, :blocks].clamp(min=0).long()

    def rows(name):  # [n, heads, tokens, dim]
        x = s[name][table].float()
        if case["kv"] == "int8":
            x = x * s[name + "_scale"][table][..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hk, blocks * block, dim)

    seq, place = _rows_of(new, s["q"].shape[0])
    q = torch.zeros(n, most, case["q_heads"], dim, device=DEVICE)
    q[seq, place] = s["q"].float()
    q = q.reshape(n, most, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(n, hk, group * most, dim)
    scores = (q @ rows("k").transpose(-1, -2)).mul_(1.0 / math.sqrt(dim)).reshape(n, hk, group, most, blocks * block)
    last = (ctx - new)[:, None] + torch.arange(most, device=DEVICE)  # the last key that a query sees
    hidden = torch.arange(blocks * block, device=DEVICE) > last[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    # a place behind a sequence's last token holds nothing: its rows are zeros
    out = (p.reshape(n, hk, group * most, -1) @ rows("v")).reshape(n, hk, group, most, dim) / total
    lse = (top + total.log())[..., 0]
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(n, most, case["q_heads"], dim)[seq, place].to(torch.bfloat16),
            "lse": lse.permute(0, 3, 1, 2).reshape(n, most, case["q_heads"])[seq, place]}


def _plain_probs(s):
    x = s["logits"] / s["case"]["temperature"]
    e = (x - x.amax(-1, keepdim=True)).exp()
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    n, most, counts = s["case"]["requests"], s["most"], s["counts_d"]
    total = s["drafts"].shape[0]
    seq, place = _rows_of(counts, total)
    first = torch.cumsum(counts, 0) - counts + torch.arange(n, device=DEVICE)  # each request's first row of the target
    x = s["drafts"].long()
    p = s["target"][first[seq] + place, x].double()
    q = s["draft"][torch.arange(total, device=DEVICE), x].double() if s["draft"] is not None else torch.ones_like(p)
    taken = torch.zeros(n, most + 1, dtype=torch.bool, device=DEVICE)
    taken[seq, place] = s["u_accept"].double() * q < p
    accepted = taken.long().cumprod(1).sum(1)
    left = s["target"][first + accepted].double()
    stopped = accepted < counts
    if total:
        at = (torch.cumsum(counts, 0) - counts + accepted).clamp(max=total - 1)
        if s["draft"] is not None:
            minus = s["draft"][at].double()
        else:
            minus = torch.zeros_like(left).scatter_(1, x[at][:, None], 1.0)
        left = torch.where(stopped[:, None], (left - minus).clamp(min=0), left)
    upto = left.cumsum(1)
    drawn = (upto > s["u_sample"].double()[:, None] * upto[:, -1:]).to(torch.int8).argmax(1)
    tokens = torch.full((n, most + 1), -1, dtype=torch.int64, device=DEVICE)
    tokens[seq, place] = torch.where(place < accepted[seq], x, -1)
    tokens[torch.arange(n, device=DEVICE), accepted] = drawn
    seq, place = _rows_of(counts + 1, total + n)
    return {"tokens": tokens[seq, place].to(torch.int32), "accepted": accepted.to(torch.int32)}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attention": _plain_attention, "probs": _plain_probs, "verify": _plain_verify}[state["case"]["op"]](state)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "append":
        new, past = _lengths(case)
        block, heads, dim = case["block"], case["heads"], case["dim"]
        need = sum(-(-(a + b) // block) for a, b in zip(new, past)) + case["seqs"]
        most = max(-(-(a + b) // block) for a, b in zip(new, past))
        tables = torch.full((1, case["seqs"], most), -1, dtype=torch.int32)
        held, free = [], 0
        for t in past:
            held.append(list(range(free, free + -(-t // block))))
            free += -(-t // block)
        for i, (a, b) in enumerate(zip(new, past)):
            more = -(-(a + b) // block) - len(held[i])
            held[i] += list(range(free, free + more))
            free += more
            tables[0, i, : len(held[i])] = torch.tensor(held[i], dtype=torch.int32)
        made = {"tables": tables, "lens": torch.tensor([[a + b for a, b in zip(new, past)]], dtype=torch.int32)}
        for name in ("k", "v"):
            pages = torch.zeros(need, block, heads, dim, dtype=torch.float64, device=DEVICE)
            old, fresh = x[name + "_past"].double().split(past), x[name].double().split(new)
            for i, ids in enumerate(held):
                rows = torch.cat([old[i], fresh[i]])
                whole = torch.zeros(len(ids) * block, heads, dim, dtype=torch.float64, device=DEVICE)
                whole[: rows.shape[0]] = rows
                pages[ids] = whole.reshape(len(ids), block, heads, dim)
            made[name] = pages.transpose(1, 2).contiguous()
        return made
    if case["op"] == "attention":
        new, ctx = _lengths(case)
        group, dim = case["q_heads"] // case["kv_heads"], case["dim"]
        if 4 * sum(m * c for m, c in zip(new, ctx)) * case["q_heads"] * dim > 6e13:
            return None
        out, lse, q0, k0 = [], [], 0, 0
        for m, c in zip(new, ctx):
            q, k, v = x["q"][q0:q0 + m].double(), x["k"][k0:k0 + c].double(), x["v"][k0:k0 + c].double()
            if case["kv"] == "int8":
                k, v = (_stored(t) for t in (k, v))
            o, z = torch.empty(m, case["q_heads"], dim, dtype=torch.float64, device=DEVICE), torch.empty(m, case["q_heads"], dtype=torch.float64, device=DEVICE)
            sees = torch.arange(c, device=DEVICE)[None] <= c - m + torch.arange(m, device=DEVICE)[:, None]
            for h in range(case["q_heads"]):
                a = torch.where(sees, q[:, h] @ k[:, h // group].T / dim ** 0.5, -math.inf)
                z[:, h] = torch.logsumexp(a, 1)
                o[:, h] = torch.exp(a - z[:, h, None]) @ v[:, h // group]
            out.append(o)
            lse.append(z)
            q0, k0 = q0 + m, k0 + c
        return {"out": torch.cat(out), "lse": torch.cat(lse)}
    if case["op"] == "probs":
        return torch.softmax(x["logits"].double() / case["temperature"], -1)
    counts = _spread(case["drafts_lo"], case["drafts_hi"], case["requests"])
    tokens, accepted, row, at = [], [], 0, 0
    for r, g in enumerate(counts):
        j, drawn = 0, []
        while j < g:
            t = int(x["drafts"][at + j])
            q = float(x["draft"][at + j, t]) if x["draft"] is not None else 1.0
            if not float(x["u_accept"][at + j]) * q < float(x["target"][row + j, t]):
                break
            drawn.append(t)
            j += 1
        left = x["target"][row + j].cpu().numpy().astype(np.float64)
        if j < g:
            minus = np.zeros_like(left)
            if x["draft"] is not None:
                minus = x["draft"][at + j].cpu().numpy().astype(np.float64)
            else:
                minus[int(x["drafts"][at + j])] = 1.0
            left = np.maximum(left - minus, 0.0)
        upto = np.cumsum(left)
        drawn.append(int(np.searchsorted(upto, float(x["u_sample"][r]) * upto[-1], side="right")))
        tokens += drawn + [-1] * (g - j)
        accepted.append(j)
        row, at = row + g + 1, at + g
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "accepted": torch.tensor(accepted, dtype=torch.int32)}


def _stored(rows):
    """What an int8 cache holds of `rows` in 64 bits: whole multiples of a scale that is kept in 32."""
    scale = rows.abs().amax(-1, keepdim=True) / 127
    scale[scale == 0] = 1
    code = rows / scale
    return torch.copysign((code.abs() + 0.5).floor(), code).clamp(-128, 127) * scale.float().double()
