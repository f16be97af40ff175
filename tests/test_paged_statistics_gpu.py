"""Statistics that are not numbers on their way through joins: a row that failed
stays one that failed, however many parts it is joined from and in whatever order.
And sequences whose tokens move from call to call under one plan's groups."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import Case  # noqa: E402
from test_paged_more_gpu import Family, joined, together  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from secure_infer_b200 import paged
    return paged


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", range(1, 9))
def test_a_logarithm_of_nan_is_kept_beside_any_others(paged, n, dtype):
    """One part's is NaN, at every place, the others' all -inf, all finite, all +inf, or some of each."""
    others = [[-math.inf], [0.5], [math.inf], [-math.inf, 0.5], [-math.inf, math.inf], [-3e38, -math.inf]]
    rows = [(at, other) for at in range(n) for other in others]
    lse = torch.tensor([[math.nan if i == at else other[i % len(other)] for i in range(n)] for at, other in rows], device="cuda")
    outs = [torch.full((len(rows), 1, 128), float(i + 1), dtype=dtype, device="cuda") for i in range(n)]
    out, got = paged.join(outs, [lse[:, i:i + 1] for i in range(n)])
    assert torch.isnan(out).all() and torch.isnan(got).all()


@pytest.mark.parametrize("n", range(1, 9))
def test_rows_that_see_nothing_and_rows_beside_failed_ones(paged, n):
    """What is -inf in every part stays so, and a NaN stays in its own row and head."""
    g = torch.Generator(device="cuda").manual_seed(n)
    outs = [torch.randn((60, 3, 128), generator=g, device="cuda").bfloat16() for _ in range(n)]
    lses = [3 * torch.randn((60, 3), generator=g, device="cuda") for _ in range(n)]
    for i, x in enumerate(lses):
        x[:20] = -math.inf
        x[20:30] = -math.inf if i else 1.0
    lses[-1][5, 1] = lses[0][40, 2] = math.nan
    failed = torch.zeros((60, 3), dtype=torch.bool, device="cuda")
    failed[5, 1] = failed[40, 2] = True
    none = torch.zeros_like(failed)
    none[:20] = True
    none &= ~failed
    out, lse = paged.join(outs, lses)
    assert torch.equal(torch.isnan(lse), failed) and torch.equal(torch.isnan(out).any(2), failed)
    assert torch.equal(lse == -math.inf, none) and (out[none] == 0).all()
    clean = [torch.where(torch.isnan(x), 0.0, x) for x in lses]
    want, want_lse, bound = joined(outs, clean)
    rest = ~failed & ~none
    assert ((out.double() - want).abs() <= bound)[rest].all()
    assert ((lse.double() - want_lse).abs() <= 2e-7 * want_lse.abs() + 1e-6)[rest].all()


def test_a_failed_call_is_seen_through_joins_in_stages(paged):
    """attend with a workspace that is down gives NaN; joined with parts that see nothing, and then with one that does,
    its rows are NaN still."""
    for lens in ([(1, 300), (3, 700)], [(200, 900), (1, 256)]):
        c = Case(paged, lens, 8, 2)
        workspace = paged.attend_workspace("cuda:0")
        workspace.view(torch.int32)[0] = 1
        failed = paged.attend(c.pages, c.chunk, c.q, return_lse=True, workspace=workspace)
        nothing = (torch.zeros_like(c.q), torch.full(c.q.shape[:2], -math.inf, device="cuda"))
        sound = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
        c.check(*sound)
        for first in ([failed, nothing], [nothing, failed], [nothing, failed, nothing]):
            stage = paged.join(*zip(*first))
            out, lse = paged.join(*zip(stage, sound))
            assert torch.isnan(out).all() and torch.isnan(lse).all()
        out, lse = paged.join(*zip(paged.join(*zip(nothing, nothing)), sound))
        assert torch.equal(out, sound[0]) and (lse - sound[1]).abs().max() <= 2e-6


@pytest.mark.parametrize("lens,groups", [([(1, 700 + 9 * i) for i in range(12)], [(12, 5)]), ([(3, 500), (1, 520), (30, 600), (1, 700)], [(4, 3)])])
def test_offsets_that_change_before_every_call(paged, lens, groups):
    """New tokens change hands between calls that follow one another without a pause, in eager mode and in a graph: every
    call's rows are those of the offsets that it was given."""
    c = Family(paged, lens, groups, 8, 2, seed=11)
    assert together(c.pages, c.chunk, c.q, c.shared)
    tokens = c.cu[-1]
    # Sequence s has a token or none, by turns; the others' tokens stay where the offsets say.
    offsets = []
    for turn in range(4):
        n = [(k if (s + turn) % 3 else 0) for s, (k, _) in enumerate(lens)]
        offsets.append([sum(n[:s]) for s in range(len(lens) + 1)])
    offsets = torch.tensor(offsets, dtype=torch.int32, device="cuda")

    def steps(outs):
        for cu, out in zip(offsets, outs):
            c.chunk.cu_q.copy_(cu)
            c.shared.update()
            paged.attend(c.pages, c.chunk, c.q, shared=c.shared, out=out)

    outs = [torch.full_like(c.q, 7.0) for _ in offsets]
    steps(outs)
    graph, again = torch.cuda.CUDAGraph(), [torch.full_like(c.q, 7.0) for _ in offsets]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        steps(again)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    all_lens, all_cu, q = c.lens, c.cu, c.q
    for cu, out, other in zip(offsets.tolist(), outs, again):
        assert (out[cu[-1]:] == 7.0).all() and torch.equal(out, other)
        c.lens, c.cu, c.q = [(b - a, kv) for a, b, (_, kv) in zip(cu, cu[1:], all_lens)], cu, q[:cu[-1]]
        c.check(out[:cu[-1]])
    assert tokens == all_cu[-1]


@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 2 ** 31 - 256, 2 ** 31 - 257, 2 ** 30, 1 << 23])
def test_trim_takes_the_sinks_that_attend_takes(paged, sinks):
    """As many sinks as a context has tokens keep all of its pages."""
    c = Family(paged, [(1, 700), (1, 650)], [(2, 4)], 8, 2)
    cache = paged.CachePages([[c.k, c.v]])
    out = paged.attend(c.pages, c.chunk, c.q, window=8, sinks=sinks)
    c.check(out)
    refs = torch.zeros(cache.pages, dtype=torch.int32, device="cuda")
    held = c.chunk.block_table[c.chunk.block_table >= 0].long()
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    t = paged.PageTables(c.chunk.block_table, c.chunk.kv_lens, refs)
    new = cache.trim(t, [0, 1], 8, sinks)
    assert all(torch.equal(a, b) for a, b in zip(new, t))
    for bad in (2 ** 31, -1):
        with pytest.raises(ValueError):
            cache.trim(t, [0, 1], 8, bad)


@pytest.mark.parametrize("lens,groups", [([(1, 700), (1, 650), (1, 643)], [(3, 4)]), ([(5, 900), (40, 1000), (1, 790)], [(3, 5)])])
def test_a_plan_outlives_lengths_that_grow(paged, lens, groups):
    """Under the same offsets a plan holds for longer sequences, eagerly and in a graph that has no update."""
    c = Family(paged, lens, groups, 8, 2, seed=12)
    whole, rows = c.lens, c.rows
    at = lambda back: ([(n, kv - back) for n, kv in whole], [[x[:kv - back] for x in r] for r, (_, kv) in zip(rows, whole)])  # noqa: E731
    c.chunk.kv_lens.sub_(3)
    c.lens, c.rows = at(3)
    c.shared.update()
    out, lse = c.run(paged)
    c.check(out, lse)
    captured, graph = torch.empty_like(c.q), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged.attend(c.pages, c.chunk, c.q, shared=c.shared, out=captured)
    for back in (2, 1, 0):
        c.chunk.kv_lens.add_(1)
        c.lens, c.rows = at(back)
        out, lse = paged.attend(c.pages, c.chunk, c.q, shared=c.shared, return_lse=True)
        c.check(out, lse)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, out)


def test_work_beyond_32_bits_with_sinks_is_refused(paged):
    """1024 sequences of one token on 8 KV heads in a table of 87380 pages: three tiles of few rows each make
    24576 * 87381 units by the usual count, which fits, and 24576 * 87382 with sinks, which does not."""
    width = 87380
    assert 24576 * (width + 1) < 2 ** 31 <= 24576 * (width + 2)
    k, v = (torch.zeros((2, 128, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cu = torch.arange(1025, dtype=torch.int32, device="cuda")
    table, none = torch.zeros((1024, width), dtype=torch.int32, device="cuda"), torch.zeros(1024, dtype=torch.int32, device="cuda")
    pages, chunk, q = paged.LayerPages(k, v), paged.Chunk(table, cu, none), torch.ones((1024, 8, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="more work than one call takes"):
        paged.attend(pages, chunk, q, window=5000, sinks=4)
    for kw in (dict(window=5000), dict(), dict(shared=paged.SharedPrefix(chunk))):
        out, lse = paged.attend(pages, chunk, q, return_lse=True, **kw)
        assert not out.any() and (lse == -math.inf).all()
    # A column less, and it fits.
    narrow = paged.Chunk(table[:, :width - 1], cu, none)
    out, lse = paged.attend(pages, narrow, q, window=5000, sinks=4, return_lse=True)
    assert not out.any() and (lse == -math.inf).all()
