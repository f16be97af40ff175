"""Several answers to one prompt whose prefix is reloaded from the host pool.

The prefix's KV blocks come back layer by layer through the authenticated reload
(``LayerwiseReloader``).  While they arrive, the prompt's last tokens run through
a small stack of attention layers with random weights: each layer appends its
keys and values to the paged cache and attends as soon as its prefix is
authentic.  The request is then forked into several answers that share the
prompt's pages, each is continued token by token, some end and give up their
pages, the cache is compacted, and the others go on.  What the answers share is
found once a step (``SharedPrefix``), and attended once for all of them where that
saves time.

    python examples/parallel_answers.py [--layers 4] [--answers 4] [--steps 6]

Needs a CUDA device and the built library.  Prints what each stage did; with
``check=True`` ``run`` compares the last step with attention over gathered keys.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from secure_infer_b200 import native_layerwise as nl, paged  # noqa: E402
from secure_infer_b200.connector import LayerwiseReloader  # noqa: E402

HEADS, KV_HEADS, DIM = 8, 2, 128


class Layer:
    """Projections of one layer of the stack."""

    def __init__(self, g):
        self.qkv = torch.randn((HEADS * DIM, (HEADS + 2 * KV_HEADS) * DIM), generator=g, device="cuda").mul_(0.03).bfloat16()
        self.out = torch.randn((HEADS * DIM, HEADS * DIM), generator=g, device="cuda").mul_(0.03).bfloat16()

    def __call__(self, x, pages, chunk, rotary, ready=None, shared=None):
        qkv = (x @ self.qkv).unflatten(1, (-1, DIM))
        q, k, v = qkv.split((HEADS, KV_HEADS, KV_HEADS), 1)
        q = paged.append(pages, chunk, q, k, v, rotary=rotary)
        if ready is not None:
            ready()   # the layer's reloaded prefix is authentic and ordered before what follows
        self.attended = paged.attend(pages, chunk, q, shared=shared)
        self.query = q
        return x + self.attended.flatten(1) @ self.out


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def run(layers=4, prefix_blocks=6, chunk_tokens=75, answers=4, steps=6, check=False, say=print):
    g = torch.Generator(device="cuda").manual_seed(1)
    pages, width = 64, prefix_blocks + 3
    session = nl.Session(0, bytes(range(16)), b"salt")
    host = [[torch.randn((prefix_blocks, 128, KV_HEADS, DIM)).bfloat16().pin_memory() for _ in range(2)] for _ in range(layers)]
    for i, pair in enumerate(host):
        for kind, t in enumerate(pair):
            nl.register_host_range(t, i, kind)
    caches = [[torch.zeros((pages, 128, KV_HEADS, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
              for _ in range(layers)]
    cache, rotary = paged.CachePages(caches), paged.Rotary(base=500000.0, device="cuda:0")
    stack, names = [Layer(g) for _ in range(layers)], [f"layer.{i}" for i in range(layers)]
    reloader = LayerwiseReloader(names, caches, host)
    try:
        # Pages for the prompt, then the prefix into the first of them.
        length = prefix_blocks * 128 + chunk_tokens
        tables = paged.PageTables(torch.full((answers, width), -1, dtype=torch.int32, device="cuda"), ints([0] * answers),
                                  ints([0] * pages))
        tables, granted = cache.reserve(tables, [0], [length])
        assert granted.tolist() == [1]
        reloader.start_load("prompt", list(range(prefix_blocks)), tables.block_table[0, :prefix_blocks].tolist())

        chunk = paged.Chunk(tables.block_table[:1], ints([0, chunk_tokens]), tables.lens[:1], max_q=chunk_tokens)
        x = torch.randn((chunk_tokens, HEADS * DIM), generator=g, device="cuda").bfloat16()
        for i, layer in enumerate(stack):
            x = layer(x, cache.layers[i], chunk, rotary, ready=lambda: reloader.wait_for_layer_load(names[i]))
        say(f"prompt: {prefix_blocks * 128} tokens reloaded, {chunk_tokens} computed over {layers} layers")

        # Every answer shares the prompt's full pages and owns a copy of its last one.
        tables, granted = cache.fork(tables, [0] * (answers - 1), list(range(1, answers)))
        assert granted.all()
        say(f"forked into {answers} answers on {int((tables.refs > 0).sum())} pages")
        alive = list(range(answers))
        x = x[-1:].repeat(answers, 1) + 0.1 * torch.randn((answers, HEADS * DIM), generator=g, device="cuda").bfloat16()
        for step in range(steps):
            if step == steps // 2 and answers > 2:
                ended = alive[1::2]
                tables = cache.free(tables, ended)
                alive = [s for s in alive if s not in ended]
                x = x[::2].contiguous()
                tables, moved, live = cache.compact(tables)
                say(f"answers {ended} ended; {int(live)} pages in use, the lowest of the cache")
            rows = ints(alive).long()
            tables, granted = cache.reserve(tables, ints(alive), tables.lens[rows] + 1)
            assert granted.all()
            chunk = paged.Chunk(tables.block_table[rows], ints(list(range(len(alive) + 1))), tables.lens[rows], max_q=1)
            shared = paged.SharedPrefix(chunk, max_common=length)   # no answer shares more than the prompt
            for i, layer in enumerate(stack):
                x = layer(x, cache.layers[i], chunk, rotary, shared=shared)
        say(f"{steps} tokens for each answer; lengths {tables.lens.tolist()}")
        off = 0.0
        if check:
            for i, layer in enumerate(stack):
                for row, s in enumerate(alive):
                    n = int(tables.lens[s])
                    k, v = (c[tables.block_table[s, :-(-n // 128)].long()].flatten(0, 1)[:n].float()
                            .repeat_interleave(HEADS // KV_HEADS, 1) for c in caches[i])
                    w = torch.softmax(torch.einsum("hd,khd->hk", layer.query[row].float(), k) * DIM ** -0.5, -1)
                    off = max(off, (torch.einsum("hk,khd->hd", w, v) - layer.attended[row].float()).abs().max().item())
                # The reloaded prefix is what the host holds, wherever compaction put it.
                where = tables.block_table[alive[0], :prefix_blocks].long()
                assert all(torch.equal(caches[i][kind][where].cpu(), host[i][kind]) for kind in range(2))
        torch.cuda.synchronize()
        return dict(tables=tables, alive=alive, output=x, off=off)
    finally:
        reloader.close()
        session.close()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--answers", type=int, default=4)
    parser.add_argument("--steps", type=int, default=6)
    args = parser.parse_args()
    print(f"largest difference from attention over gathered keys: "
          f"{run(args.layers, answers=args.answers, steps=args.steps, check=True)['off']:.4f}")
