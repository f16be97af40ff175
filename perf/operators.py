"""Cases and plain forms of the paged-cache operators.

Three operators work on the paged KV cache that reloads fill: ``append`` rotates a chunk's queries and keys and
writes its keys and values into their pages, ``attend`` is the attention of the chunk over the pages, and
``CachePages`` forks, frees and compacts pages.  A layer's cache is ``[pages, 128 tokens, KV heads, 128]``.

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
    def attend(name, heads, kv_heads, chunks, q, kv, decodes=0, decode_kv=0, idle=0, window=0, lse=False, dtype="bf16"):
        return dict(name=name, op="attend", heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=kv,
                    decodes=decodes, decode_kv=decode_kv, idle=idle, window=window, lse=lse, dtype=dtype, lens=7)

    def append(name, heads, kv_heads, chunks, q, kv, decodes, axes, dtype="bf16"):
        return dict(name=name, op="append", heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=kv,
                    decodes=decodes, decode_kv=kv, idle=0, axes=axes, base=500000.0, dtype=dtype, lens=7)

    return [
        # One request answering token by token right after a short prompt (Llama-3-8B heads): latency alone.
        attend("decode, 1 sequence of 200", 32, 8, 0, 0, 0, decodes=1, decode_kv=200),
        # A serving batch of single tokens over ragged contexts, one slot of it idle (Qwen2.5-7B heads, groups of 7).
        attend("decode, 48 up to 8192, group 7", 28, 4, 0, 0, 0, decodes=47, decode_kv=8192, idle=1),
        # One long document on one GPU of a 70B model at TP = 8: one KV head, the context has to be split.
        attend("decode, 1 of 131072, 1 KV head", 8, 1, 0, 0, 0, decodes=1, decode_kv=131072),
        # The suffix of a request whose 6144-token prefix was reloaded (Llama-3-8B heads).
        attend("chunk of 512 after 6144", 32, 8, 1, 512, 6656),
        # Chunked prefill beside running requests: a chunk of odd length and single tokens in one call, with statistics.
        attend("mixed, 333 and 15 singles", 32, 8, 1, 333, 2500, decodes=15, decode_kv=4000, lse=True),
        # Short drafts to verify (speculative decoding), sliding window, fp16.
        attend("drafts of 5, window 1000, fp16", 32, 8, 24, 5, 4096, window=1000, dtype="fp16"),
        # A long prompt's last chunk: bound by the tensor cores.
        attend("chunk of 4096 in 20480", 32, 8, 1, 4096, 20480),
        # Single tokens of a batch: positions on one axis.
        append("append 16 single tokens", 32, 8, 0, 0, 4096, 16, 1),
        # A large ragged prefill step with time, height and width positions.
        append("append 8000, three axes", 28, 4, 5, 1777, 6144, 3, 3),
        # Parallel answers to one prompt: the partial last page is copied in every layer (70B shard, 80 layers of 1 head).
        dict(name="fork 24 children", op="fork", layers=80, kv_heads=1, pages=320, seqs=64, width=64, n=24, kv=900, lens=7),
        # Requests that ended: their pages go back, in a cache of many sequences.
        dict(name="free 300 of 512 sequences", op="free", layers=1, kv_heads=1, pages=20000, seqs=512, width=256, n=300, kv=9000, lens=7),
        # Compaction after many requests ended: live pages move down (Llama-3-8B, 32 layers of 8 heads).
        dict(name="compact 32 of 96 pages", op="compact", layers=32, kv_heads=8, pages=96, seqs=32, width=16, n=32, kv=256, lens=7),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["attend", "attend", "attend", "append", "fork", "free", "compact"])
    lens = rng.randrange(1 << 30)
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (8, 1), (16, 4), (7, 1), (4, 4), (64, 8), (12, 2)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attend":
        chunks = rng.choice([0, 0, 1, 1, log(1, 8), log(2, 24)])
        q = log(1, 4096 if chunks == 1 else 600) if chunks else 0
        decodes = log(1, 64) if not chunks else rng.choice([0, 0, log(1, 24)])
        kv = (q + log(1, 16000)) if chunks else 0
        decode_kv = log(1, 131072 if decodes == 1 else 9000) if decodes else 0
        # The plain form's padded scores stay within 1.5 G values, its gathered keys within 1 G.
        idle = rng.choice([0, 0, 1, 3])
        while chunks and (decodes + chunks + idle) * heads * q * max(kv, decode_kv) > 1.5e9:
            decodes, chunks, idle, q = decodes // 2, max(1, chunks // 2), idle // 2, max(1, q * 3 // 4)
            kv = max(q, kv * 3 // 4)
            decode_kv = max(1, decode_kv * 3 // 4) if decodes else 0
        while (decodes + chunks + idle) * kv_heads * DIM * max(kv, decode_kv) > 1e9:
            decodes, kv, decode_kv = max(1 - min(1, chunks), decodes // 2), max(q, kv // 2), decode_kv // 2
        return dict(op=op, heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=kv, decodes=decodes,
                    decode_kv=decode_kv, idle=idle, window=rng.choice([0, 0, 0, log(1, 3000)]),
                    lse=rng.random() < 0.25, dtype=dtype, lens=lens)
    if op == "append":
        chunks, decodes = rng.choice([(0, log(1, 256)), (1, 0), (log(1, 8), log(1, 32))])
        q = log(1, 12000 // max(1, chunks)) if chunks else 0
        return dict(op=op, heads=heads, kv_heads=kv_heads, chunks=chunks, q=q, kv=q + log(1, 4000), decodes=decodes,
                    decode_kv=log(1, 4000), idle=rng.choice([0, 0, 2]), axes=rng.choice([1, 1, 3]),
                    base=rng.choice([10000.0, 500000.0, 1000000.0]), dtype=dtype, lens=lens)
    if op == "free":
        seqs, kv = log(1, 1024), log(1, 12000)
        return dict(op=op, layers=1, kv_heads=1, pages=seqs * -(-kv // PAGE) + rng.randrange(1, 3000), seqs=seqs,
                    width=-(-kv // PAGE) + rng.randrange(0, 65), n=rng.randint(1, seqs), kv=kv, lens=lens)
    layers, kv_heads = rng.choice([(32, 8), (28, 4), (80, 1), (5, 2), (1, 8)])
    budget = int(1.6e9) // (layers * 2 * PAGE * kv_heads * DIM * 2)
    pages = log(12, max(13, min(2000, budget)))
    if op == "fork":
        seqs = log(4, 256)
        kv = max(1, min(log(1, 3000), PAGE * (pages // 2)))
        return dict(op=op, layers=layers, kv_heads=kv_heads, pages=pages, seqs=seqs, width=-(-kv // PAGE) + rng.randrange(0, 9),
                    n=max(1, min(seqs // 2, pages // 4)), kv=kv, lens=lens)
    n = log(1, max(1, pages // 3))
    return dict(op=op, layers=layers, kv_heads=kv_heads, pages=pages, seqs=rng.randint(1, 64), width=rng.randint(8, 40),
                n=n, kv=PAGE * rng.randint(1, 4), lens=lens)


def lengths(case):
    """Tokens in the chunk and in all of each sequence: the chunks first, then single tokens, then idle slots."""
    r = random.Random(case["lens"])
    q, kv = [], []
    for i in range(case["chunks"]):
        q.append(case["q"] if i == 0 else r.randint(max(1, case["q"] // 2), case["q"]))
        kv.append(case["kv"] if i == 0 else r.randint(q[-1], max(q[-1], case["kv"])))
    for i in range(case["decodes"]):
        q.append(1)
        kv.append(case["decode_kv"] if i == 0 else r.randint(1, case["decode_kv"]))
    return q + [0] * case["idle"], kv + [0] * case["idle"]


def used(tokens):
    return -(-tokens // PAGE)


def visible(q, kv, window):
    """(query, key) pairs of one sequence that the causal mask and the window leave."""
    first = kv - q
    return sum(min(first + i + 1, window) if window else first + i + 1 for i in range(q))


def held(case):
    """Lengths of the sequences in a table: the first n empty (a fork's children), the others up to case["kv"]."""
    r = random.Random(case["lens"])
    empty = case["n"] if case["op"] == "fork" else 0
    left = case["pages"] - empty
    lens = [0] * empty
    for i in range(case["seqs"] - empty):
        t = case["kv"] if i == 0 else r.randint(1, case["kv"])
        t = min(t, left * PAGE)
        left -= used(t)
        lens.append(t)
    return lens


def parents(case):
    r = random.Random(case["lens"] + 1)
    return [r.randrange(case["n"], case["seqs"]) for _ in range(case["n"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if case["op"] in ("attend", "append"):
        dtype = TYPES[case["dtype"]]
        q_lens, kv_lens = lengths(case)
        total, pages = sum(q_lens), sum(used(t) for t in kv_lens) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        width = max(used(t) for t in kv_lens) + 1
        # Sequence s owns the next used(kv) pages of a shuffled order; entries past them are -1.
        starts = ints([sum(used(t) for t in kv_lens[:i]) for i in range(len(kv_lens))])
        col = torch.arange(width, device="cuda")
        own_pages = ints([used(t) for t in kv_lens])
        at = (starts[:, None] + col).clamp(max=pages - 1).long()
        table = torch.where(col < own_pages[:, None], order[at], -1).to(torch.int32)
        shape = (pages, PAGE, case["kv_heads"], DIM)
        cache = [torch.randn(shape, generator=g, device="cuda", dtype=dtype) for _ in range(2)]
        state = dict(case=case, k_cache=cache[0], v_cache=cache[1], table=table, kv=ints(kv_lens),
                     cu=ints([sum(q_lens[:i]) for i in range(len(q_lens) + 1)]), max_q=max(q_lens), total=total,
                     width=width)
        if case["op"] == "attend":
            # Queries of real layers are larger than N(0, 1): a softmax with some peaks.
            state["q"] = 2 * torch.randn((total, case["heads"], DIM), generator=g, device="cuda", dtype=dtype)
            # What a page holds past its sequence's length was never written.
            token = (torch.arange(width * PAGE, device="cuda") >= state["kv"][:, None]).reshape(len(kv_lens), width, PAGE)
            sl = token & (table >= 0)[:, :, None]
            page = table.clamp(min=0).long()[:, :, None].expand_as(sl)[sl]
            slot = torch.arange(PAGE, device="cuda").expand_as(sl)[sl]
            for c in cache:
                c[page, slot] = float("nan")
        else:
            # Queries, keys and values as one projection leaves them: slices of one row.
            h, n = case["heads"], case["kv_heads"]
            qkv = torch.randn((total, h + 2 * n, DIM), generator=g, device="cuda", dtype=dtype)
            state["q"], state["k"], state["v"] = qkv[:, :h], qkv[:, h:h + n], qkv[:, h + n:]
            if case["axes"] == 1:
                state["sections"] = (64,)
                seq, row = token_rows(state["cu"], total)
                first = state["kv"] - (state["cu"][1:] - state["cu"][:-1])
                state["positions"] = (first[seq] + row).to(torch.int32)[None].contiguous()
            else:
                # Frames of a grid after some text: time, height and width of every token.
                state["sections"] = (16, 24, 24)
                t = torch.arange(total, device="cuda") + torch.randint(0, 4000, (1,), generator=g, device="cuda")
                state["positions"] = torch.stack((t // 480, t // 24 % 20 + t // 480, t % 24 + t // 480)).to(torch.int32)
        if own:
            from secure_infer_b200 import paged

            state["pages"] = paged.LayerPages(state["k_cache"], state["v_cache"])
            state["chunk"] = paged.Chunk(table, state["cu"], state["kv"], max_q=state["max_q"])
            if case["op"] == "append":
                state["rotary"] = paged.Rotary(base=case["base"], sections=state["sections"], device="cuda")
        return state

    shape = (case["layers"], 2, case["pages"], PAGE, case["kv_heads"], DIM)
    cache = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    lens = held(case)
    order = torch.randperm(case["pages"], generator=g, device="cuda").tolist()
    if case["op"] == "compact":
        # Of `live` pages, n lie at or above `live` and have to move; the sequences share the live pages.
        live = case["pages"] - case["n"] - (case["pages"] - 2 * case["n"]) // 3
        r = random.Random(seed)
        below, above = list(range(live)), list(range(live, case["pages"]))
        n = min(case["n"], len(above))
        r.shuffle(below)
        r.shuffle(above)
        owned = below[n:] + above[:n]
        r.shuffle(owned)
        rows, refs = [[] for _ in range(case["seqs"])], [0] * case["pages"]
        for i, p in enumerate(owned):
            if len(rows[i % case["seqs"]]) < case["width"]:
                rows[i % case["seqs"]].append(p)
            refs[p] += 1
        for row in rows[1:]:  # a prefix page that several sequences share
            if len(row) < case["width"] and rows[0]:
                row.insert(0, rows[0][0])
                refs[rows[0][0]] += 1
        lens = [len(row) * PAGE - (5 if row else 0) for row in rows]
    else:
        rows, refs, k = [], [0] * case["pages"], 0
        for t in lens:
            rows.append(order[k:k + used(t)])
            k += used(t)
            for p in rows[-1]:
                refs[p] = 1
    table = ints([row + [-1] * (case["width"] - len(row)) for row in rows])
    state = dict(case=case, cache=cache, table=table, lens=ints(lens), refs=ints(refs))
    if case["op"] == "fork":
        state["from"], state["to"] = ints(parents(case)), ints(list(range(case["n"])))
    if case["op"] == "free":
        r = random.Random(seed)
        state["ended"] = ints(r.sample(range(case["seqs"]), case["n"]))
    if own:
        from secure_infer_b200 import paged

        state["pages"] = paged.CachePages([[c[0], c[1]] for c in cache])
        state["tables"] = paged.PageTables(state["table"], state["lens"], state["refs"])
    return state


def run(state):
    case = state["case"]
    if own:
        from secure_infer_b200 import paged

        if case["op"] == "attend":
            return paged.attend(state["pages"], state["chunk"], state["q"], window=case["window"], return_lse=case["lse"])
        if case["op"] == "append":
            q = paged.append(state["pages"], state["chunk"], state["q"], state["k"], state["v"],
                             rotary=state["rotary"], positions=state["positions"])
            return q, state["k_cache"], state["v_cache"]
        if case["op"] == "fork":
            t, granted = state["pages"].fork(state["tables"], state["from"], state["to"])
            return t.block_table, t.lens, t.refs, granted, state["cache"]
        if case["op"] == "free":
            t = state["pages"].free(state["tables"], state["ended"])
            return t.block_table, t.lens, t.refs
        t, moved, live = state["pages"].compact(state["tables"])
        return t.block_table, t.lens, t.refs, moved, live, state["cache"]
    return PLAIN[case["op"]](state)


def token_rows(cu, total):
    """Sequence of each token of a chunk, and its row there."""
    token = torch.arange(total, device=cu.device)
    seq = torch.searchsorted(cu[1:].long(), token, right=True)
    return seq, token - cu[seq]


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
    if case["window"]:
        seen = seen & (key > at - case["window"])
    v = v.masked_fill((key >= kv[:, None])[:, :, None, None], 0.0)
    s = torch.einsum("sqhgd,skhd->shgqk", x, k) * DIM ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("shgqk,skhd->shgqd", p, v) / total
    o = o.masked_fill(~seen.any(-1)[:, None, None, :, None], 0.0)
    seq, r = token_rows(cu, state["total"])
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, r].to(dtype)
    if not case["lse"]:
        return out
    lse = (m + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).flatten(2, 3)
    return out, lse[seq, r]


def plain_append(state):
    case, kv, cu = state["case"], state["kv"], state["cu"]
    dtype = state["q"].dtype
    axis = torch.repeat_interleave(torch.arange(len(state["sections"])), torch.tensor(state["sections"])).tolist()
    freq = case["base"] ** (-torch.arange(64, device="cuda", dtype=torch.float32) / 64)
    angle = (state["positions"][axis].float().T * freq)[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)

    def rotated(x):
        a, b = x[..., :64].float(), x[..., 64:].float()
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(dtype)

    seq, row = token_rows(cu, state["total"])
    at = kv[seq] - (cu[1:] - cu[:-1])[seq] + row
    page, slot = state["table"][seq, at // PAGE].long(), at % PAGE
    state["k_cache"][page, slot] = rotated(state["k"])
    state["v_cache"][page, slot] = state["v"]
    return rotated(state["q"]), state["k_cache"], state["v_cache"]


def plain_fork(state):
    table, lens, refs, cache = state["table"].clone(), state["lens"].clone(), state["refs"].clone(), state["cache"]
    parent, child = state["from"].long(), state["to"].long()
    n = lens[parent]
    need, full = (n % PAGE > 0).int(), (n // PAGE)[:, None]
    free = torch.argsort((refs != 0).int(), stable=True).int()  # free pages first, lowest ids first
    place = torch.cumsum(need, 0) - need
    granted = ((lens[child] == 0) & ((place + need <= (refs == 0).sum()) | (need == 0))).int()
    new = free[place.clamp(max=len(free) - 1)]
    copied = (granted * need) > 0
    col = torch.arange(table.shape[1], device="cuda")
    rows = torch.where(col < full, table[parent], torch.where((col == full) & copied[:, None], new[:, None], -1))
    old = table[parent, (n // PAGE).clamp(max=table.shape[1] - 1).long()]
    src, dst = old[copied].long(), new[copied].long()
    cache[:, :, dst] = cache[:, :, src]
    ok = granted.bool()
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), ((rows >= 0) & ok[:, None]).int().flatten())
    table[child] = torch.where(ok[:, None], rows, table[child]).int()
    lens[child] = torch.where(ok, n, lens[child])
    return table, lens, refs, granted, cache


def plain_free(state):
    table, lens, refs, ended = state["table"].clone(), state["lens"].clone(), state["refs"].clone(), state["ended"].long()
    rows = table[ended]
    mine = torch.arange(table.shape[1], device="cuda") < ((lens[ended] + PAGE - 1) // PAGE)[:, None]
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), -mine.int().flatten())
    table[ended] = -1
    lens[ended] = 0
    return table, lens, refs


def plain_compact(state):
    table, refs, cache = state["table"], state["refs"], state["cache"]
    page = torch.arange(refs.shape[0], device="cuda")
    alive = refs > 0
    live = alive.sum()
    src, dst = torch.nonzero(alive & (page >= live))[:, 0], torch.nonzero(~alive & (page < live))[:, 0]
    moved = torch.where(alive, page, -1)
    moved[src] = dst
    cache[:, :, dst] = cache[:, :, src]
    counts = torch.zeros_like(refs)
    counts[moved[alive]] = refs[alive]
    mine = torch.arange(table.shape[1], device="cuda") < ((state["lens"] + PAGE - 1) // PAGE)[:, None]
    table = torch.where(mine, moved[table.clamp(min=0).long()], -1)
    return table.int(), state["lens"].clone(), counts, moved.int(), live.int().reshape(1), cache


PLAIN = dict(attend=plain_attend, append=plain_append, fork=plain_fork, free=plain_free, compact=plain_compact)


def work(case):
    if case["op"] in ("attend", "append"):
        q_lens, kv_lens = lengths(case)
        rows = sum(q_lens)
        if case["op"] == "append":
            moved = rows * (case["heads"] + 2 * case["kv_heads"]) * DIM * 2 * 2
            return {"bytes": moved + 4 * rows * case["axes"], "flops": rows * (case["heads"] + case["kv_heads"]) * DIM * 3}
        read = sum(min(kv, case["window"] + q - 1) if case["window"] else kv for q, kv in zip(q_lens, kv_lens) if q)
        pairs = sum(visible(q, kv, case["window"]) for q, kv in zip(q_lens, kv_lens))
        moved = 2 * rows * case["heads"] * DIM * 2 + 2 * read * case["kv_heads"] * DIM * 2
        return {"bytes": moved + 4 * rows * case["heads"] * case["lse"], "flops": 4 * pairs * case["heads"] * DIM}
    tables = 2 * 4 * (case["seqs"] * (case["width"] + 1) + case["pages"])
    page = case["layers"] * 2 * PAGE * case["kv_heads"] * DIM * 2
    if case["op"] == "fork":
        lens = held(case)
        return {"bytes": tables + 2 * page * sum(lens[p] % PAGE > 0 for p in parents(case)), "flops": 0}
    if case["op"] == "free":
        return {"bytes": tables, "flops": 0}
    live = case["pages"] - case["n"] - (case["pages"] - 2 * case["n"]) // 3
    return {"bytes": tables + 4 * case["pages"] + 2 * page * min(case["n"], case["pages"] - live), "flops": 0}


def exact(case, seed):
    """From the definitions, in 64 bits, one sequence and one head at a time."""
    if case["op"] not in ("attend", "append"):
        return None
    state = prepare(case, seed)
    q_lens, kv_lens = lengths(case)
    out = state["q"].double()
    if case["op"] == "append":
        pair = torch.arange(64, dtype=torch.float64, device="cuda")
        freq = torch.exp(-pair / 64 * math.log(case["base"]))
        bounds = [sum(state["sections"][:i + 1]) for i in range(len(state["sections"]))]
        axis = [sum(i >= b for b in bounds) for i in range(64)]
        angle = torch.stack([state["positions"][axis[i]].double() * freq[i] for i in range(64)], 1)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def rotated(x):
            z = torch.complex(x[..., :64].double(), x[..., 64:].double()) * turn
            return torch.cat((z.real, z.imag), -1)

        k_cache, v_cache = state["k_cache"].double(), state["v_cache"].double()
        k, table, token = rotated(state["k"]), state["table"].tolist(), 0
        for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
            for first in range((kv - n) // PAGE * PAGE, kv if n else 0, PAGE):  # page by page
                a, b = max(first, kv - n), min(first + PAGE, kv)
                k_cache[table[s][first // PAGE], a - first:b - first] = k[token:token + b - a]
                v_cache[table[s][first // PAGE], a - first:b - first] = state["v"][token:token + b - a].double()
                token += b - a
        return rotated(state["q"]), k_cache, v_cache
    group = case["heads"] // case["kv_heads"]
    lse = torch.full((state["total"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    token = 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        if not n:
            continue
        where = state["table"][s, :used(kv)].long()
        position = torch.arange(kv - n, kv, device="cuda")[:, None]
        key = torch.arange(kv, device="cuda")[None]
        hidden = key > position
        if case["window"]:
            hidden = hidden | (position - key >= case["window"])
        for h in range(case["heads"]):
            k = state["k_cache"][where, :, h // group].reshape(-1, DIM)[:kv].double()
            v = state["v_cache"][where, :, h // group].reshape(-1, DIM)[:kv].double()
            a = state["q"][token:token + n, h].double() @ k.T / math.sqrt(DIM)
            a.masked_fill_(hidden, -math.inf)
            lse[token:token + n, h] = torch.logsumexp(a, 1)
            out[token:token + n, h] = torch.softmax(a, 1) @ v
        token += n
    return (out, lse) if case["lse"] else out
