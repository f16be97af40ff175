"""Cases and plain forms of the paged cache's operators for long requests and for batches with one prompt.

``attend`` with a sliding window and sinks sees the first tokens of a sequence and its last ones; ``trim`` gives back
the pages between them.  ``attend`` of a batch that shares a prefix reads the pages that its sequences have in common
once for all of them.  ``join`` makes attention over parts of the keys into attention over all.  A layer's cache is
``[pages, 128 tokens, KV heads, 128]``.

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is true, through
``secure_infer_b200.paged``.  Sequence lengths come from the case alone, values and page orders from the seed.
"""
import math
import random

import torch

own = False

PAGE = 128
DIM = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    def sinks(name, heads, kv_heads, chunks, q, kv, window, sinks, decodes=0, decode_kv=0, idle=0, lse=False, dtype="bf16"):
        return dict(name=name, op="sinks", heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=kv, decodes=decodes,
                    decode_kv=decode_kv, idle=idle, window=window, sinks=sinks, lse=lse, dtype=dtype, lens=7)

    def shared(name, heads, kv_heads, groups, members, prompt, rest, q, lse=False, dtype="bf16"):
        return dict(name=name, op="shared", heads=heads, kv_heads=kv_heads, groups=groups, members=members,
                    prompt=prompt, rest=rest, q=q, lse=lse, dtype=dtype, lens=7)

    return [
        # One long-running request, token by token, a short window: latency alone (Llama-3-8B heads).
        sinks("sinks, 1 sequence of 700", 32, 8, 0, 0, 0, 512, 4, decodes=1, decode_kv=700),
        # A serving batch of endless streams, ragged, one slot idle (Qwen2.5-7B heads, groups of 7).
        sinks("sinks, 47 up to 16384, group 7", 28, 4, 0, 0, 0, 4000, 4, decodes=47, decode_kv=16384, idle=1),
        # A chunk of odd length beside running requests, with statistics.
        sinks("sinks, 777 and 3 singles, fp16", 32, 8, 1, 777, 9000, 1024, 100, decodes=3, decode_kv=5000, lse=True, dtype="fp16"),
        # A long prompt's chunk under a window: bound by the tensor cores.
        sinks("sinks, chunk of 4096 in 16384", 32, 8, 1, 4096, 16384, 4096, 128),
        # After a step of a few requests: the pages that fell out of their windows go back.
        dict(name="trim 8 sequences", op="trim", pages=700, seqs=8, width=80, n=8, kv=9000, window=1000, sinks=4, lens=7),
        # The same in a cache of many sequences.
        dict(name="trim 300 of 512 sequences", op="trim", pages=20000, seqs=512, width=256, n=300, kv=9000, window=2048, sinks=64, lens=7),
        # Two answers to a short prompt: latency alone.
        shared("shared, 2 answers to 600", 32, 8, 1, 2, 600, 40, 1),
        # Many answers to a long prompt, token by token.
        shared("shared, 48 answers to 8192", 32, 8, 1, 48, 8192, 1000, 1),
        # Drafts of several answers to several documents, one KV head of a 70B model at TP = 8, with statistics.
        shared("shared, 4 x 6 drafts of 5, fp16", 8, 1, 4, 6, 30000, 700, 5, lse=True, dtype="fp16"),
        # Questions on one document: each a ragged chunk of its own after the same pages.
        shared("shared, 5 questions up to 300", 28, 4, 1, 5, 6144, 300, 300),
        # Single tokens' attention over two sets of keys, joined.
        dict(name="join 2 parts of 16 tokens", op="join", parts=2, tokens=16, heads=32, dtype="bf16"),
        # A large prefill step, attended in three parts.
        dict(name="join 3 parts of 8000 tokens", op="join", parts=3, tokens=8000, heads=28, dtype="bf16"),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["sinks", "sinks", "sinks", "shared", "shared", "shared", "join", "trim"])
    lens = rng.randrange(1 << 30)
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (8, 1), (16, 4), (7, 1), (4, 4), (64, 8), (12, 2)])
    dtype, lse = rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.25
    if op == "sinks":
        chunks = rng.choice([0, 0, 1, 1, log(1, 8), log(2, 24)])
        q = log(1, 4096 if chunks == 1 else 600) if chunks else 0
        decodes = log(1, 64) if not chunks else rng.choice([0, 0, log(1, 24)])
        kv = (q + log(1, 12000)) if chunks else 0
        decode_kv = log(1, 65536 if decodes == 1 else 9000) if decodes else 0
        idle = rng.choice([0, 0, 1, 3])
        # The plain form's padded scores stay within 1.2 G values, its gathered keys within 0.8 G.
        while chunks and (decodes + chunks + idle) * heads * q * max(kv, decode_kv) > 1.2e9:
            decodes, chunks, idle, q = decodes // 2, max(1, chunks // 2), idle // 2, max(1, q * 3 // 4)
            kv = max(q, kv * 3 // 4)
            decode_kv = max(1, decode_kv * 3 // 4) if decodes else 0
        while (decodes + chunks + idle) * kv_heads * DIM * max(kv, decode_kv) > 8e8:
            decodes, kv, decode_kv = max(1 - min(1, chunks), decodes // 2), max(q, kv // 2), decode_kv // 2
        return dict(op=op, heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=kv, decodes=decodes,
                    decode_kv=decode_kv, idle=idle, window=log(1, 6000), sinks=rng.choice([0, log(1, 8), log(1, 1000)]),
                    lse=lse, dtype=dtype, lens=lens)
    if op == "shared":
        groups, members = rng.choice([(1, log(2, 64)), (1, log(2, 64)), (log(2, 6), log(2, 10))])
        q, prompt = rng.choice([1, 1, log(1, 8), log(1, 400)]), log(100, 32000)
        rest = q + rng.choice([0, log(1, 1500)])
        while groups * members * heads * q * (prompt + rest) > 1.2e9:
            q, prompt = max(1, q // 2), max(100, prompt * 3 // 4)
        while groups * members * kv_heads * DIM * (prompt + rest) > 8e8:
            groups, members = max(1, groups - 1), max(2, members * 3 // 4)
            prompt = max(100, prompt * 3 // 4)
        return dict(op=op, heads=heads, kv_heads=kv_heads, groups=groups, members=members, prompt=prompt, rest=rest, q=q,
                    lse=lse, dtype=dtype, lens=lens)
    if op == "join":
        return dict(op=op, parts=rng.randint(2, 6), tokens=log(1, 9000), heads=heads, dtype=dtype)
    seqs, kv = log(1, 1024), log(1, 12000)
    return dict(op=op, pages=seqs * used(kv) + rng.randrange(1, 2000), seqs=seqs, width=used(kv) + rng.randrange(0, 65),
                n=rng.randint(1, seqs), kv=kv, window=log(1, 6000), sinks=rng.choice([0, log(1, 8), log(1, 1000)]), lens=lens)


def used(tokens):
    return -(-tokens // PAGE)


def lengths(case):
    """New tokens and all tokens of each sequence, and how many pages from its first it shares with its group."""
    r = random.Random(case["lens"])
    q, kv, common = [], [], []
    if case["op"] == "shared":
        for g in range(case["groups"]):
            prompt = case["prompt"] if g == 0 else r.randint(max(1, case["prompt"] // 3), case["prompt"])
            for i in range(case["members"]):
                # Single tokens and drafts are of one length, longer chunks ragged.
                q.append(case["q"] if case["q"] <= 8 or i == 0 else r.randint(1, case["q"]))
                kv.append(prompt + (case["rest"] if i == 0 else r.randint(q[-1], case["rest"])))
                common.append(prompt // PAGE)
        return q, kv, common
    for i in range(case["chunks"]):
        q.append(case["q"] if i == 0 else r.randint(max(1, case["q"] // 2), case["q"]))
        kv.append(case["kv"] if i == 0 else r.randint(q[-1], max(q[-1], case["kv"])))
    for i in range(case["decodes"]):
        q.append(1)
        kv.append(case["decode_kv"] if i == 0 else r.randint(1, case["decode_kv"]))
    q, kv = q + [0] * case["idle"], kv + [0] * case["idle"]
    return q, kv, [0] * len(q)


def held(case):
    """Lengths of the sequences in a table."""
    r = random.Random(case["lens"])
    left, lens = case["pages"], []
    for i in range(case["seqs"]):
        lens.append(min(case["kv"] if i == 0 else r.randint(1, case["kv"]), left * PAGE))
        left -= used(lens[-1])
    return lens


def trimmed(case, tokens):
    """Pages of a sequence of `tokens` that lie between its sinks and the next token's window."""
    return max(0, (tokens - case["window"] + 1) // PAGE - used(case["sinks"]))


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "join":
        dtype, rows = TYPES[case["dtype"]], (case["tokens"], case["heads"])
        outs = [torch.randn((*rows, DIM), generator=g, device="cuda", dtype=dtype) for _ in range(case["parts"])]
        # Logarithms of sums over some hundred or thousand keys; a few rows see no key of a part.
        lses = [6 + 2 * torch.randn(rows, generator=g, device="cuda") for _ in range(case["parts"])]
        for o, x in zip(outs, lses):
            none = torch.rand(rows, generator=g, device="cuda") < 0.02
            x.masked_fill_(none, -math.inf)
            o.masked_fill_(none[..., None], 0.0)
        return dict(case=case, outs=outs, lses=lses)
    if case["op"] == "trim":
        order = torch.randperm(case["pages"], generator=g, device="cuda").tolist()
        lens, rows, refs, at = held(case), [], [0] * case["pages"], 0
        for t in lens:
            rows.append(order[at:at + used(t)])
            at += used(t)
            for p in rows[-1]:
                refs[p] = 1
        for row in rows[1:]:   # a prompt's first page that several sequences share
            if row and rows[0] and used(case["kv"]) > 2:
                refs[row[0]] -= 1
                row[0] = rows[0][0]
                refs[row[0]] += 1
        ended = random.Random(seed).sample(range(case["seqs"]), case["n"])
        state = dict(case=case, table=ints([row + [-1] * (case["width"] - len(row)) for row in rows]), lens=ints(lens),
                     refs=ints(refs), named=ints(ended))
        if own:
            from secure_infer_b200 import paged

            cache = torch.zeros((2, case["pages"], PAGE, 1, DIM), device="cuda", dtype=torch.bfloat16)
            state["pages"] = paged.CachePages([[cache[0], cache[1]]])
            state["tables"] = paged.PageTables(state["table"], state["lens"], state["refs"])
        return state

    dtype = TYPES[case["dtype"]]
    q_lens, kv_lens, common = lengths(case)
    seqs, total, width = len(q_lens), sum(q_lens), max(used(t) for t in kv_lens) + 1
    n, kv = ints(q_lens), ints(kv_lens)
    col = torch.arange(width, device="cuda")
    if case["op"] == "sinks":
        # Pages that no token from the first new one on sees were given back.
        lo = (kv - n - case["window"] + 1)[:, None]
        mine = (col < used_of(kv)[:, None]) & ((PAGE * (col + 1) > lo) | (PAGE * col < case["sinks"]))
    else:
        mine = col < used_of(kv)[:, None]
    # A group's first sequence owns the pages that the others share.
    first = torch.arange(seqs, device="cuda") // case.get("members", 1) * case.get("members", 1)
    borrowed = (col < ints(common)[:, None]) & (first != torch.arange(seqs, device="cuda"))[:, None]
    owned = mine & ~borrowed
    pages = int(owned.sum()) + 3
    order = torch.randperm(pages, generator=g, device="cuda")
    table = torch.full((seqs, width), -1, device="cuda")
    table[owned] = order[:pages - 3]
    table = torch.where(borrowed, table[first], table).to(torch.int32)
    shape = (pages, PAGE, case["kv_heads"], DIM)
    cache = [torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(2)]
    # What a page holds past its sequence's length was never written.
    token = (torch.arange(width * PAGE, device="cuda") >= kv[:, None]).reshape(seqs, width, PAGE) & owned[:, :, None]
    page, slot = table.long()[:, :, None].expand_as(token)[token], torch.arange(PAGE, device="cuda").expand_as(token)[token]
    for c in cache:
        c[page, slot] = float("nan")
    # Queries of real layers are larger than N(0, 1): a softmax with some peaks.
    q = 2 * torch.randn((total, case["heads"], DIM), generator=g, device="cuda", dtype=dtype)
    state = dict(case=case, k_cache=cache[0], v_cache=cache[1], table=table, kv=kv, q=q, total=total, max_q=max(q_lens),
                 cu=ints([sum(q_lens[:i]) for i in range(seqs + 1)]), window=case.get("window", 0), sinks=case.get("sinks", 0))
    if own:
        from secure_infer_b200 import paged

        state["pages"] = paged.LayerPages(*cache)
        state["chunk"] = paged.Chunk(table, state["cu"], kv, max_q=state["max_q"])
        if case["op"] == "shared":
            # Found once a step, for all its layers.
            state["shared"] = paged.SharedPrefix(state["chunk"], ints(list(range(0, seqs + 1, case["members"]))))
    return state


def used_of(tokens):
    return (tokens + PAGE - 1) // PAGE


def run(state):
    case = state["case"]
    if own:
        from secure_infer_b200 import paged

        if case["op"] == "sinks":
            return paged.attend(state["pages"], state["chunk"], state["q"], window=case["window"], sinks=case["sinks"],
                                return_lse=case["lse"])
        if case["op"] == "shared":
            return paged.attend(state["pages"], state["chunk"], state["q"], shared=state["shared"], return_lse=case["lse"])
        if case["op"] == "join":
            return paged.join(state["outs"], state["lses"])
        t = state["pages"].trim(state["tables"], state["named"], window=case["window"], sinks=case["sinks"])
        return t.block_table, t.lens, t.refs
    return PLAIN[case["op"]](state)


def plain_attend(state):
    case, kv, cu = state["case"], state["kv"], state["cu"]
    q, dtype = state["q"], state["q"].dtype
    h = case["kv_heads"]
    table = state["table"].clamp(min=0).long()
    k = state["k_cache"][table].float().flatten(1, 2)
    v = state["v_cache"][table].float().flatten(1, 2)
    n_q = cu[1:] - cu[:-1]
    row, key = torch.arange(state["max_q"], device="cuda"), torch.arange(k.shape[1], device="cuda")
    x = q[(cu[:-1, None] + row).clamp(max=state["total"] - 1)].float().unflatten(2, (h, -1))
    at = ((kv - n_q)[:, None] + row)[:, :, None]
    seen = (key <= at) & (key < kv[:, None, None])
    if state["window"]:
        seen = seen & ((key > at - state["window"]) | (key < state["sinks"]))
    v = v.masked_fill(~seen.any(1)[:, :, None, None], 0.0)
    s = torch.einsum("sqhgd,skhd->shgqk", x, k) * DIM ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("shgqk,skhd->shgqd", p, v) / total
    o = o.masked_fill(~seen.any(-1)[:, None, None, :, None], 0.0)
    token = torch.arange(state["total"], device="cuda")
    seq = torch.searchsorted(cu[1:].long(), token, right=True)
    r = token - cu[seq]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, r].to(dtype)
    if not case["lse"]:
        return out
    lse = (m + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).flatten(2, 3)
    return out, lse[seq, r]


def plain_join(state):
    lse = torch.stack(state["lses"])
    m = lse.amax(0).clamp(min=torch.finfo(torch.float32).min)
    w = torch.exp(lse - m)
    total = w.sum(0)
    o = (w[..., None] * torch.stack(state["outs"]).float()).sum(0) / total[..., None]
    o = o.masked_fill((total == 0)[..., None], 0.0)
    return o.to(state["outs"][0].dtype), m + torch.log(total)


def plain_trim(state):
    case, lens = state["case"], state["lens"]
    table, refs, named = state["table"].clone(), state["refs"].clone(), state["named"].long()
    rows, col = table[named], torch.arange(table.shape[1], device="cuda")
    gone = (PAGE * col >= case["sinks"]) & (PAGE * (col + 1) <= (lens[named] - case["window"] + 1)[:, None]) & (rows >= 0)
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), -gone.int().flatten())
    table[named] = rows.masked_fill(gone, -1)
    return table, lens.clone(), refs


PLAIN = dict(sinks=plain_attend, shared=plain_attend, join=plain_join, trim=plain_trim)


def work(case):
    if case["op"] == "join":
        rows = case["tokens"] * case["heads"]
        return {"bytes": (case["parts"] + 1) * rows * (2 * DIM + 4), "flops": 2 * case["parts"] * rows * DIM}
    if case["op"] == "trim":
        return {"bytes": 2 * 4 * (case["seqs"] * (case["width"] + 1) + case["pages"]), "flops": 0}
    q_lens, kv_lens, common = lengths(case)
    rows = sum(q_lens)
    w, s, pairs, read = case.get("window", 0), case.get("sinks", 0), 0, 0
    for i, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if not n:
            continue
        if w:
            lo = max(0, kv - n - w + 1)
            read += kv - lo + min(s, lo)
            pairs += sum(min(p + 1, w + min(s, max(0, p - w + 1))) for p in range(kv - n, kv))
        else:
            read += kv - (PAGE * common[i] if i % case["members"] else 0)
            pairs += sum(range(kv - n + 1, kv + 1))
    moved = 2 * rows * case["heads"] * DIM * 2 + 2 * read * case["kv_heads"] * DIM * 2
    return {"bytes": moved + 4 * rows * case["heads"] * case["lse"], "flops": 4 * pairs * case["heads"] * DIM}


def exact(case, seed):
    """From the definitions, in 64 bits, one sequence and one head at a time."""
    if case["op"] == "trim":
        return None
    state = prepare(case, seed)
    if case["op"] == "join":
        lse = torch.logsumexp(torch.stack([x.double() for x in state["lses"]]), 0)
        out = torch.zeros(state["outs"][0].shape, dtype=torch.float64, device="cuda")
        for o, x in zip(state["outs"], state["lses"]):
            weight = torch.exp(x.double() - lse)
            out += torch.where(torch.isfinite(x), weight, 0.0)[..., None] * o.double()
        return out, lse
    q_lens, kv_lens, _ = lengths(case)
    group = case["heads"] // case["kv_heads"]
    out = state["q"].double()
    lse = torch.full((state["total"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    token = 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if not n:
            continue
        position = torch.arange(kv - n, kv, device="cuda")[:, None]
        # The keys that its page table still has.
        where = state["table"][s, :used(kv)].long()
        key = torch.arange(kv, device="cuda")[(where >= 0).repeat_interleave(PAGE)[:kv]]
        page, slot = where[key // PAGE], key % PAGE
        hidden = key[None] > position
        if case["op"] == "sinks":
            hidden = hidden | ((position - key >= case["window"]) & (key >= case["sinks"]))
        for h in range(case["heads"]):
            k, v = (state[c][page, slot, h // group].double() for c in ("k_cache", "v_cache"))
            a = state["q"][token:token + n, h].double() @ k.T / math.sqrt(DIM)
            a.masked_fill_(hidden, -math.inf)
            lse[token:token + n, h] = torch.logsumexp(a, 1)
            out[token:token + n, h] = torch.softmax(a, 1) @ v
        token += n
    return (out, lse) if case["lse"] else out
