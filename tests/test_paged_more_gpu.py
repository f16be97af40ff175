"""Attention with sinks behind a window, with shared prefixes, the joining of
parts and the trimming of pages, against their definitions in 64 bits.

Bounds.  Attention: as in test_paged_gpu.py, whose cases these build on: a weight
is rounded once to the cache's type (relative to the largest weight of its part,
which is at most the row's largest after joining), an output once.  ``join``
rounds its outputs once; its weights e^(lse_i - lse) are off by 2^-23 for the
exponential, by 2^-24 of an argument below 40 times log2(e) (4e-6), and by as much
for the sum: 1e-5 of sum w |o|.  Its logarithm is off by 2^-23 of itself and 1e-6
for the sum."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_gpu import EDGES, EPS, Case, consistent, model_of  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from secure_infer_b200 import paged
    return paged


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Seen(Case):
    """A case whose expected rows may see sinks as well."""

    def expected(self, causal=True, window=0, scale=None, sinks=0):
        if not sinks:
            return super().expected(causal, window, scale)
        scale = 128 ** -0.5 if scale is None else scale
        eps = EPS[self.dtype]
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        for s, (n, kv) in enumerate(self.lens):
            if n == 0 or kv == 0:
                continue
            k, v = (x.double().repeat_interleave(self.group, 1) for x in self.rows[s])
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None]
            seen = (key <= pos) & ((key > pos - window) | (key < sinks))
            some = seen.any(0)                     # what no row sees takes no part, whatever it holds
            k, v, seen = k[some], v[some], seen[:, some]
            x = torch.einsum("qhd,khd->hqk", self.q[self.cu[s]:self.cu[s + 1]].double(), k) * scale
            x = x.masked_fill(~seen, -math.inf)
            any_key = seen.any(1)
            w = torch.softmax(x, -1).masked_fill(~seen, 0.0)
            bad = ~torch.isfinite(v)
            o = torch.einsum("hqk,khd->qhd", w, v.masked_fill(bad, 0.0))
            for value in (math.inf, -math.inf, math.nan):
                at = torch.isnan(v) if math.isnan(value) else v == value
                if at.any():
                    o = torch.where(torch.einsum("qk,khd->qhd", seen.double(), at.double()) > 0, o + value, o)
            mass = torch.einsum("hqk,khd->qhd", w, v.abs().masked_fill(bad, 0.0))
            tail = kv * 2.0 ** -25 * v.abs().masked_fill(bad, 0.0).amax() if self.dtype == torch.float16 and v.numel() else 0.0
            rows = slice(self.cu[s], self.cu[s + 1])
            out[rows] = torch.where(any_key[:, None, None], o, 0.0)
            bound[rows] = eps * o.abs() + (eps + 2e-4) * mass + tail + 1e-7
            lse[rows] = torch.where(any_key[:, None], torch.logsumexp(x, -1).T, -math.inf)
        return out, lse, bound

    def attend(self, paged, window, sinks, **kw):
        return paged.attend(self.pages, self.chunk, self.q, window=window, sinks=sinks, return_lse=True, **kw)

    def hide(self, s, window, sinks, value=math.nan):
        """Write `value` over every key that no row of sequence s sees, and give back its whole pages; -> pages given back."""
        n, kv = self.lens[s]
        lo, gone = max(0, kv - n - window + 1), 0
        for p in range(-(-kv // 128)):
            page = self.table[s, p].item()
            for slot in range(max(0, sinks - 128 * p), min(128, lo - 128 * p)):
                self.k[page, slot] = value
                self.v[page, slot] = value
            if 128 * p >= sinks and 128 * (p + 1) <= lo:
                self.table[s, p] = -1 - p
                gone += 1
        return gone


# -------------------------------------------------------------------- sinks

@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (8, 1), (40, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window,sinks", [(1, 1), (5, 4), (100, 16), (128, 128), (200, 129), (300, 260)])
def test_single_tokens_with_sinks(paged, heads, kv_heads, dtype, window, sinks):
    c = Seen(paged, [(1, n) for n in EDGES], heads, kv_heads, dtype)
    out, lse = c.attend(paged, window, sinks)
    c.check(out, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("window,sinks", [(1, 1), (3, 20), (64, 4), (127, 128), (128, 127), (129, 33), (500, 400)])
@pytest.mark.parametrize("lens", [[(2, 2), (5, 700), (5, 5), (3, 129)], [(16, 900), (8, 131)], [(200, 900), (70, 70)],
                                  [(300, 1500), (1, 1000), (2, 40), (0, 9)], [(520, 2000)]])
def test_drafts_and_chunks_with_sinks(paged, window, sinks, lens):
    c = Seen(paged, lens, 8, 2, seed=window)
    out, lse = c.attend(paged, window, sinks)
    c.check(out, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (3, 3), (160, 1), (7, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_layouts_with_sinks(paged, heads, kv_heads, dtype):
    c = Seen(paged, [(129, 1100), (1, 700), (4, 600)], heads, kv_heads, dtype, seed=3)
    out, lse = c.attend(paged, 150, 10)
    c.check(out, lse, window=150, sinks=10)


@pytest.mark.parametrize("lens", [[(1, 1000), (6, 1000), (150, 1000)], [(1, 130), (3, 200), (40, 250)], [(1, 20000)],
                                  [(300, 3000)]])
@pytest.mark.parametrize("window,sinks", [(100, 4), (60, 100), (200, 128), (33, 140)])
def test_what_lies_between_sinks_and_window_may_hold_anything(paged, lens, window, sinks):
    """Whole pages there have been given away, parts of a page beside sinks or window hold what they hold."""
    c = Seen(paged, lens, 8, 2)
    want, want_lse = c.attend(paged, window, sinks)
    c.check(want, want_lse, window=window, sinks=sinks)
    for s in range(len(lens)):
        c.hide(s, window, sinks)
    table = c.table.cuda()
    c.chunk.block_table.copy_(table)
    for value in (math.nan, math.inf):
        out, lse = c.attend(paged, window, sinks)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,kv", [(1, 700), (5, 700), (16, 300), (140, 600), (300, 320), (60, 60)])
def test_odd_values_among_sinks_and_window(paged, n, kv, value):
    """A value reaches the rows that see its key and no others: at a sink all rows behind it, in the window some."""
    window, sinks = 50, 40
    for key in sorted({3, sinks - 1, sinks, max(0, kv - n - 20), max(0, kv - n // 2 - 1), kv - 1}):
        c = Seen(paged, [(n, kv)], 4, 2, seed=5)
        c.set_row(0, key, 1, v=value)
        out, lse = c.attend(paged, window, sinks)
        c.check(out, lse, window=window, sinks=sinks)


def test_a_sinks_key_of_nan_makes_its_rows_nan(paged):
    c = Seen(paged, [(3, 500), (200, 700), (200, 200)], 4, 2, seed=6)
    for s in range(3):
        c.set_row(s, 2, 0, k=math.nan)
    out, _ = c.attend(paged, 64, 4)
    want, _, bound = c.expected(window=64, sinks=4)
    seen = torch.ones(out.shape[0], dtype=torch.bool, device="cuda")
    seen[203:205] = False    # the third sequence's tokens 0 and 1
    assert torch.isnan(out[seen][:, :2]).all()
    assert ((out.double() - want).abs() <= bound)[~seen].all() and ((out.double() - want).abs() <= bound)[:, 2:].all()


@pytest.mark.parametrize("lens", [[(1, 300), (1, 900)], [(6, 900), (200, 1200)]])
def test_sinks_and_windows_as_long_as_a_context(paged, lens):
    """Sinks or a window as long as a context leave the causal order; no sinks leave the window."""
    c = Seen(paged, lens, 8, 2)
    for window, sinks in ((1, 5000), (2 ** 31 - 1, 2 ** 31 - 1), (7, 900), (900, 1)):
        out, lse = c.attend(paged, window, sinks)
        c.check(out, lse, window=window, sinks=sinks)
        if max(window, sinks) >= 1200:
            c.check(out, lse)
    out, lse = c.attend(paged, 70, 0)
    c.check(out, lse, window=70)


@pytest.mark.parametrize("lens", [[(0, 0), (1, 40), (0, 300), (1, 128)], [(3, 0), (1, 0)], [(10, 4), (200, 50), (1, 300)]])
def test_rows_that_see_nothing_with_sinks(paged, lens):
    c = Seen(paged, lens, 8, 2)
    out, lse = c.attend(paged, 20, 7, out=torch.full_like(c.q, math.nan))
    c.check(out, lse, window=20, sinks=7)


@pytest.mark.parametrize("lens,window,sinks", [([(1, 60000)], 20000, 9000), ([(7, 30000)], 9000, 300), ([(100, 20000)], 6000, 2000),
                                               ([(1, 9000)] * 5 + [(400, 9000)], 3000, 130)])
def test_long_contexts_with_sinks_repeat(paged, lens, window, sinks):
    c = Seen(paged, lens, 8, 1)
    out, lse = c.attend(paged, window, sinks)
    c.check(out, lse, window=window, sinks=sinks)
    for _ in range(10):
        again, again_lse = c.attend(paged, window, sinks)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_many_sequences_of_both_kinds_with_sinks(paged):
    """More sequences than a block has threads, chunks among single tokens and drafts; the same bits again."""
    c = Seen(paged, [(40 if i % 7 == 0 else 1 + i % 4, 40 + (i * 37) % 500) for i in range(1400)], 8, 2)
    out, lse = c.attend(paged, 60, 5)
    c.check(out, lse, window=60, sinks=5)
    again, again_lse = c.attend(paged, 60, 5)
    assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("lens", [[(1, 20000)] * 30 + [(30, 50)], [(2000, 2100)] + [(1, 40)] * 3, [(24, 300), (25, 300), (3, 9000)]])
def test_one_kind_has_most_of_the_work(paged, lens):
    c = Seen(paged, lens, 4, 4)
    out, lse = c.attend(paged, 9000, 8)
    c.check(out, lse, window=9000, sinks=8)


@pytest.mark.parametrize("layout", ["heads", "joint"])
def test_layouts_with_sinks(paged, layout):
    c = Seen(paged, [(1, 700), (3, 300), (150, 800)], 12, 2, layout=layout)
    qkv = torch.randn((c.q.shape[0], 16, 128), device="cuda").to(c.dtype)
    qkv[:, 2:14] = c.q
    out, lse = paged.attend(c.pages, c.chunk, qkv[:, 2:14], window=90, sinks=30, return_lse=True, scale=-0.05)
    c.check(out, lse, window=90, sinks=30, scale=-0.05)


def test_rows_whose_sinks_are_minus_infinity(paged):
    """Sinks with scores of minus infinity have no weight; where the window's are too there is no softmax."""
    for lens in ([(1, 900)], [(5, 700)], [(200, 1000)]):
        c = Seen(paged, lens, 4, 2, seed=7)
        c.q[:, :, 0] = 1.0
        for j in range(4):
            c.set_row(0, j, 0, k=torch.tensor([-math.inf] + [0.0] * 127, device="cuda", dtype=c.dtype))
        out, lse = c.attend(paged, 64, 4)
        c.check(out, lse, window=64, sinks=4)
        n, kv = lens[0]
        for j in range(kv - n - 64, kv):
            c.set_row(0, j, 0, k=torch.tensor([-math.inf] + [0.0] * 127, device="cuda", dtype=c.dtype))
        out, _ = c.attend(paged, 64, 4)
        assert torch.isnan(out[:, :2]).all() and torch.isfinite(out[:, 2:]).all()


# ------------------------------------------------------------ shared prefixes

def together(pages, chunk, q, shared):
    """Whether a call attends what groups have in common together."""
    from secure_infer_b200 import _native
    ct = _native.ct
    c = _native.Chunk.from_buffer_copy(chunk._c)
    c.tokens = q.shape[0]
    o = _native.AttendOptions(shared._plan.data_ptr(), None, shared.groups, shared.max_common)
    return _native.lib().secure_infer_attend_parts(pages._address, ct.addressof(c), q.shape[1], ct.addressof(o)) > 0


class Family(Seen):
    """Groups of sequences whose first pages are the same.  groups: (sequences, pages in common)."""

    def __init__(self, paged, lens, groups, heads, kv_heads, dtype=torch.bfloat16, seed=0, **kw):
        super().__init__(paged, lens, heads, kv_heads, dtype, seed, **kw)
        self.bounds, s0 = [0], 0
        for n, pages in groups:
            long = [s for s in range(s0, s0 + n) if lens[s][1] >= 128 * pages]   # the others cannot hold what is common
            for s in long[1:]:
                self.table[s, :pages] = self.table[long[0], :pages]
                for x, y in zip(self.rows[s], self.rows[long[0]]):
                    x[:128 * pages] = y[:128 * pages]
            s0 += n
            self.bounds.append(s0)
        # In a wide table groups are attended together however small they are.
        table = torch.full((len(lens), 1 << 16), -1, dtype=torch.int32, device="cuda")
        table[:, :self.table.shape[1]] = self.table.cuda()
        self.chunk = paged.Chunk(table, self.chunk.cu_q, self.chunk.kv_lens, max_q=max(n for n, _ in lens))
        self.shared = paged.SharedPrefix(self.chunk, ints(self.bounds))

    def tokens(self):
        """Of each sequence, what the groups have in common."""
        common = [0] * len(self.lens)
        for a, b in zip(self.bounds, self.bounds[1:]):
            rows = [s for s in range(a, b) if self.lens[s][0]]
            if len(rows) < 2:
                continue
            most = min(max(0, self.lens[s][1] - self.lens[s][0]) // 128 for s in rows)
            same = (self.table[rows] == self.table[rows[:1]]).all(0).tolist()
            for s in range(a, b):
                common[s] = 128 * next((i for i in range(most) if not same[i]), most)
        return common

    def saves(self):
        """Whether rows of a page are fewer tiles together than apart."""
        time = lambda rows: 4 * -(-rows // 8) if rows <= 24 else 4 if rows <= 128 else 7 * -(-rows // 256)  # noqa: E731
        tokens, groups = self.cu[-1], self.shared.groups
        seqs = min(len(self.lens), tokens)
        return seqs * time(-(-tokens // seqs) * self.group) > groups * time(-(-tokens // groups) * self.group)

    def run(self, paged, **kw):
        assert self.shared.tokens.tolist() == self.tokens()
        assert together(self.pages, self.chunk, self.q, self.shared) or not self.saves()
        return paged.attend(self.pages, self.chunk, self.q, shared=self.shared, return_lse=True, **kw)


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (8, 1), (4, 4), (40, 2), (160, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,groups", [
    ([(1, 300), (1, 257)], [(2, 2)]),
    ([(1, 130 + 41 * i) for i in range(9)], [(9, 1)]),
    ([(1, 1300 + 7 * i) for i in range(40)], [(40, 10)]),
    ([(1, 500), (1, 600), (1, 2000), (1, 1900), (1, 1930), (1, 77)], [(2, 3), (3, 12), (1, 0)]),
])
def test_answers_to_one_prompt(paged, heads, kv_heads, dtype, lens, groups):
    c = Family(paged, lens, groups, heads, kv_heads, dtype)
    out, lse = c.run(paged)
    c.check(out, lse)


@pytest.mark.parametrize("lens,groups", [
    ([(5, 900), (5, 903), (5, 850)], [(3, 6)]),                               # drafts: 20 rows a sequence, 60 a prefix
    ([(100, 700), (33, 640), (250, 900)], [(3, 4)]),                          # questions on one document
    ([(1, 700), (300, 1500), (2, 800), (1, 650)], [(4, 5)]),                  # all kinds
    ([(300, 1000), (300, 1000), (1, 400), (1, 402), (7, 4000), (7, 4001)], [(2, 4), (2, 3), (2, 30)]),
    ([(600, 1600), (700, 1900)], [(2, 7)]),                                   # tiles of both sequences' rows
    ([(0, 0), (1, 500), (0, 900), (1, 520), (0, 0)], [(5, 3)]),               # idle slots among them
    ([(1, 128), (1, 129), (1, 256)], [(3, 1)]),                               # a page is common only if it lies before all new tokens
    ([(200, 128), (3, 1), (1, 300)], [(3, 1)]),                               # more new tokens than tokens
])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_chunks_and_edges(paged, lens, groups, causal):
    c = Family(paged, lens, groups, 8, 2, seed=2)
    out, lse = c.run(paged, causal=causal, out=torch.full_like(c.q, math.nan))
    c.check(out, lse, causal=causal)


def test_prefixes_as_they_are_found(paged):
    """What is common goes by the tables: nothing, some pages, all before the new tokens; groups in any form."""
    lens = [(1, 700), (1, 650), (1, 900), (2, 700), (1, 640), (1, 130)]
    c = Family(paged, lens, [(2, 5), (3, 4), (1, 1)], 8, 2)
    assert c.tokens() == [640, 640, 512, 512, 512, 0] and c.shared.tokens.tolist() == c.tokens()
    whole = paged.SharedPrefix(c.chunk)
    assert whole.tokens.tolist() == [0] * 6 and whole.groups == 1
    out, lse = paged.attend(c.pages, c.chunk, c.q, shared=whole, return_lse=True)
    c.check(out, lse)
    assert torch.equal(out, paged.attend(c.pages, c.chunk, c.q))
    # Sequences outside of every group, groups that are empty, out of order or out of range.
    for bounds, want in (([1, 2], [0] * 6), ([2, 5], [0, 0, 512, 512, 512, 0]), ([0, 2, 2, 5], c.tokens()),
                         ([0, 5, 2, 6], [0] * 6), ([-7, 2, 99], [640, 640, 0, 0, 0, 0]), ([4, 2, 5, 9], [0] * 6),
                         ([0, 1, 2, 3, 4, 5, 6], [0] * 6)):
        found = paged.SharedPrefix(c.chunk, ints(bounds))
        assert found.tokens.tolist() == want, bounds
        out, lse = paged.attend(c.pages, c.chunk, c.q, shared=found, return_lse=True)
        c.check(out, lse)


@pytest.mark.parametrize("seqs", [300, 1500])
def test_groups_of_many_sequences(paged, seqs):
    """More sequences and groups than a block has threads, and one group of all."""
    lens = [(int(i % 5 != 3), 140 + (i * 37) % 300) for i in range(seqs)]
    c = Family(paged, lens, [(3, 1)] * (seqs // 3), 4, 2, seed=seqs)
    out, lse = c.run(paged)
    c.check(out, lse)
    c = Family(paged, lens, [(seqs, 1)], 4, 2, seed=seqs)
    out, lse = c.run(paged)
    c.check(out, lse)


@pytest.mark.parametrize("lens,groups,heads", [([(1, 20000 + i) for i in range(3)], [(3, 156)], 8),
                                               ([(1, 9000 + 300 * i) for i in range(12)], [(12, 70)], 8),
                                               ([(5, 9000)] * 6 + [(200, 3000)] * 2, [(6, 60), (2, 20)], 16)])
def test_long_prefixes_repeat(paged, lens, groups, heads):
    """Prefixes and own keys that are cut over many CTAs: the same bits whoever finishes last."""
    c = Family(paged, lens, groups, heads, 1)
    out, lse = paged.attend(c.pages, c.chunk, c.q, shared=c.shared, return_lse=True)
    c.check(out, lse)
    out, lse = c.run(paged)
    c.check(out, lse)
    for _ in range(10):
        again, again_lse = paged.attend(c.pages, c.chunk, c.q, shared=c.shared, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,groups", [([(1, 700), (1, 690)], [(2, 4)]), ([(140, 700), (3, 690), (1, 600)], [(3, 3)])])
def test_odd_values_with_a_shared_prefix(paged, value, lens, groups):
    """A value in a common page reaches every row, one in a sequence's own the rows of it that see its key."""
    for s, key in ((0, 5), (0, 650), (1, 688)):
        c = Family(paged, lens, groups, 4, 2, seed=4)
        c.set_row(s, key, 1, v=value)
        if key < 128:
            for other in range(1, len(lens)):
                c.rows[other][1][key, 1] = value
        out, lse = c.run(paged)
        c.check(out, lse)


def test_scores_of_minus_infinity_in_a_shared_prefix(paged):
    """A prefix without weight leaves the rest; where the rest has none either there is no softmax."""
    low = torch.tensor([-math.inf] + [0.0] * 127, device="cuda", dtype=torch.bfloat16)
    for lens in ([(1, 300), (1, 290)], [(150, 500), (150, 480)]):
        c = Family(paged, lens, [(2, 2)], 4, 2, seed=7)
        c.q[:, :, 0] = 1.0
        for j in range(256):
            c.set_row(0, j, 0, k=low)
            c.rows[1][0][j, 0] = low
        out, lse = c.run(paged)
        c.check(out, lse)
        for j in range(256, lens[0][1]):
            c.set_row(0, j, 0, k=low)
        out, _ = c.run(paged)
        n = lens[0][0]
        assert torch.isnan(out[:n, :2]).all() and torch.isfinite(out[n:]).all() and torch.isfinite(out[:, 2:]).all()


@pytest.mark.parametrize("lens,groups,shares", [([(1, 5200 + 9 * i) for i in range(30)], [(30, 40)], True),
                                                ([(5, 9000)] * 8 + [(5, 9100)] * 8, [(8, 70), (8, 70)], True),
                                                ([(1, 300), (1, 310)], [(2, 2)], False), ([(300, 900), (280, 900)], [(2, 4)], False)])
def test_sharing_where_it_saves_time(paged, lens, groups, shares):
    """Narrow tables, and wide ones with a bound on what is common, leave the choice to the sizes."""
    c = Family(paged, lens, groups, 32, 8, seed=8)
    narrow = paged.Chunk(c.chunk.block_table[:, :c.table.shape[1]], c.chunk.cu_q, c.chunk.kv_lens, max_q=c.chunk._c.max_q)
    for chunk, most in ((narrow, None), (c.chunk, 128 * max(n for _, n in groups))):
        shared = paged.SharedPrefix(chunk, ints(c.bounds), max_common=most)
        assert shared.tokens.tolist() == c.tokens() and together(c.pages, chunk, c.q, shared) == shares
        out, lse = paged.attend(c.pages, chunk, c.q, shared=shared, return_lse=True)
        c.check(out, lse)
        if not shares:
            assert torch.equal(out, paged.attend(c.pages, chunk, c.q))


def test_tokens_of_nobody_stay_with_a_shared_prefix(paged):
    c = Family(paged, [(1, 300), (1, 290), (40, 400)], [(3, 2)], 8, 2)
    q = torch.cat((c.q, torch.full((9, 8, 128), math.nan, dtype=c.dtype, device="cuda")))
    out = torch.full_like(q, 7.0)
    paged.attend(c.pages, c.chunk, q, shared=c.shared, out=out)
    c.check(out[:42])
    assert (out[42:] == 7.0).all()


def test_plans_follow_the_chunk_in_a_graph(paged):
    """A captured update and attend follow lengths and tables; without an update more tokens may come behind a prefix."""
    c = Family(paged, [(1, 700), (1, 650), (1, 640)], [(3, 4)], 8, 2)
    out = torch.empty_like(c.q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.shared.update()
        for _ in range(2):
            paged.attend(c.pages, c.chunk, c.q, shared=c.shared, out=out)
    for step in range(4):
        if step == 2:   # another table: one page is common
            c.table[2, 1:4] = c.table[1, 1:4] = c.table[0, 1:4]
            c.table[2, 1] = c.table[2, 4]
            c.chunk.block_table[:, :c.table.shape[1]].copy_(c.table)
            for which, cache in enumerate((c.k, c.v)):
                for i in range(4):
                    c.rows[2][which][128 * i:128 * (i + 1)] = cache[c.table[2, i].item()]
            # (Page 4 of sequence 2 holds 128 tokens: 640 in all.)
        c.chunk.kv_lens.sub_(1)
        c.lens = [(n, kv - 1) for n, kv in c.lens]
        c.rows = [[x[:kv] for x in r] for r, (_, kv) in zip(c.rows, c.lens)]
        graph.replay()
        torch.cuda.synchronize()
        assert c.shared.tokens.tolist() == c.tokens()
        c.check(out)


def test_stale_plans_stay_within_bounds(paged):
    """A plan for other lengths is an error of the caller's, which reads and writes nothing outside."""
    c = Family(paged, [(1, 700), (1, 650), (40, 640)], [(3, 4)], 8, 2)
    out = torch.zeros_like(c.q)
    for lens in ([0, 0, 0], [100, 600, 41], [1 << 30, -5, 512]):
        c.chunk.kv_lens.copy_(ints(lens))
        paged.attend(c.pages, c.chunk, c.q, shared=c.shared, out=out)
    c.chunk.kv_lens.copy_(ints([700, 650, 640]))
    c.chunk.cu_q.copy_(ints([5, 2, 900, -3]))
    paged.attend(c.pages, c.chunk, c.q, shared=c.shared, out=out)
    paged.SharedPrefix(c.chunk, ints([0, 3]))
    c.chunk.cu_q.copy_(ints(c.cu))
    out, lse = c.run(paged)
    c.check(out, lse)


@pytest.mark.parametrize("lens,groups", [([(1, 3000), (1, 2900), (1, 2950)], [(3, 20)]), ([(100, 2000), (90, 1900), (1, 1800)], [(3, 12)])])
def test_shared_calls_on_streams_and_in_graphs(paged, lens, groups):
    """Eager calls on one stream beside replays on another: their workspaces and parts are their own."""
    a, b = Family(paged, lens, groups, 8, 1, seed=1), Family(paged, lens, groups, 8, 1, seed=2)
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        want_a, want_b = (paged.attend(c.pages, c.chunk, c.q, shared=c.shared) for c in (a, b))
    first.synchronize()
    a.check(want_a)
    b.check(want_b)
    out, graph = torch.empty_like(b.q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=first):
        for _ in range(3):
            paged.attend(b.pages, b.chunk, b.q, shared=b.shared, out=out)
    got = []
    for _ in range(20):
        with torch.cuda.stream(second):
            graph.replay()
        with torch.cuda.stream(first):
            got += [paged.attend(a.pages, a.chunk, a.q, shared=a.shared) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_a) for x in got) and torch.equal(out, want_b)


@pytest.mark.parametrize("how", ["sinks", "shared"])
def test_a_workspace_that_is_down(paged, how):
    """Rows are NaN in every form of the call until the status has been read."""
    for lens, groups in (([(1, 300), (3, 320)], [(2, 2)]), ([(200, 700), (150, 900), (1, 640)], [(3, 3)]), ([(1, 9000)] * 3, [(3, 60)]),
                         ([(100, 9000)] * 2, [(2, 60)])):
        c = Family(paged, lens, groups, 8, 1)
        kw = dict(window=64, sinks=5) if how == "sinks" else dict(shared=c.shared)
        workspace = paged.attend_workspace("cuda:0")
        workspace.view(torch.int32)[0] = 1
        for _ in range(2):
            out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True, workspace=workspace, **kw)
            assert torch.isnan(out).all() and torch.isnan(lse).all()
        assert paged.attend_status(workspace) == 1
        out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True, workspace=workspace, **kw)
        c.check(out, lse, **({} if how == "shared" else kw))
        assert paged.attend_status(workspace) == 0 and not workspace[:4096].any()


# --------------------------------------------------------------------- join

def joined(outs, lses):
    """In 64 bits, and its bound."""
    x = torch.stack([l.double() for l in lses])
    lse = torch.logsumexp(x, 0)
    w = torch.where(x == -math.inf, 0.0, torch.exp(x - lse))
    o = torch.stack([o.double() for o in outs])
    o = torch.where((x == -math.inf)[..., None], 0.0, o)
    out = (w[..., None] * o).sum(0)
    return out, lse, EPS[outs[0].dtype] * out.abs() + 1e-5 * (w[..., None] * o.abs()).sum(0) + 1e-7


def check_join(paged, outs, lses, **kw):
    want, want_lse, bound = joined(outs, lses)
    out, lse = paged.join(outs, lses, **kw)
    assert out.dtype == outs[0].dtype and lse.dtype == torch.float32
    assert ((out.double() - want).abs() <= bound).all()
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert ((lse.double() - want_lse).abs() <= 2e-7 * want_lse.abs() + 1e-6)[~empty].all()
    return out, lse


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 7), (3, 28), (17, 32), (1000, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_join(paged, n, tokens, heads, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    outs = [torch.randn((tokens, heads, 128), generator=g, device="cuda").to(dtype) for _ in range(n)]
    lses = [5 * torch.randn((tokens, heads), generator=g, device="cuda") for _ in range(n)]
    check_join(paged, outs, lses)
    for i, x in enumerate(lses):   # parts of which a row sees nothing, and rows that see nothing at all
        x.view(-1)[i % 3::3] = -math.inf
    outs[0].view(-1, 128)[::3] = math.nan
    out, lse = check_join(paged, outs, lses)
    if n > 3 or tokens * heads > 3:
        assert torch.isfinite(out).all()


def test_join_strides_and_places(paged):
    dtype = torch.bfloat16
    wide = torch.randn((50, 20, 128), device="cuda").to(dtype)
    outs = [wide[:, 3:9], wide[:, 9:15], torch.randn((6, 50, 128), device="cuda").to(dtype).transpose(0, 1)]
    lses = [torch.randn((6, 50), device="cuda").T, torch.randn((50, 12), device="cuda")[:, ::2], torch.randn(50, device="cuda")[:, None].expand(50, 6)]
    want, _ = check_join(paged, outs, lses)
    given = torch.empty((50, 6, 128), dtype=dtype, device="cuda")
    assert paged.join(outs, lses, out=given)[0] is not None and torch.equal(given, want)
    # Over one of the parts.
    dense = [o.contiguous() for o in outs]
    got, _ = paged.join(dense, lses, out=dense[1])
    assert torch.equal(dense[1], want) and got.data_ptr() == dense[1].data_ptr()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        other = paged.join(outs, lses)[0]
    side.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.join(outs, lses, out=given)
    given.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(given, want)
    assert paged.join([wide[:0]], [torch.empty((0, 20), device="cuda")])[0].shape == (0, 20, 128)


def test_join_of_odd_statistics(paged):
    """NaN stays NaN, and sums far apart or far from zero lose nothing."""
    outs = [torch.full((4, 2, 128), float(i + 1), dtype=torch.float16, device="cuda") for i in range(2)]
    lses = [torch.zeros((4, 2), device="cuda") for _ in range(2)]
    lses[0][0], lses[1][1], lses[0][2], lses[1][2], lses[0][3], lses[1][3] = math.nan, math.nan, -3e4, 3e4, -1e5, -1e5
    out, lse = paged.join(outs, lses)
    assert torch.isnan(out[:2]).all() and torch.isnan(lse[:2]).all()
    assert (out[2] == 2).all() and (lse[2] == 3e4).all() and (out[3] == 1.5).all()
    # Two sums of e^-100000 make log 2 more, rounded to the nearest of 32 bits.
    assert (lse[3] == torch.tensor(-1e5 + math.log(2), dtype=torch.float32)).all()


@pytest.mark.parametrize("lens", [[(1, 700), (1, 300)], [(5, 800)], [(200, 900), (1, 640)]])
def test_parts_of_the_keys_make_the_whole(paged, lens):
    """Attention over a context's first pages and over the rest, joined."""
    c = Seen(paged, lens, 8, 2)
    first = paged.Chunk(c.chunk.block_table[:, :2], c.chunk.cu_q, ints([256 if n else 0 for n, _ in lens]), max_q=c.chunk._c.max_q)
    rest = paged.Chunk(c.chunk.block_table[:, 2:], c.chunk.cu_q, c.chunk.kv_lens - 256, max_q=c.chunk._c.max_q)
    parts = [paged.attend(c.pages, first, c.q, causal=False, return_lse=True), paged.attend(c.pages, rest, c.q, return_lse=True)]
    out, lse = paged.join(*zip(*parts))
    want, want_lse, bound = c.expected()
    # Each part was rounded once more.
    assert ((out.double() - want).abs() <= bound + EPS[c.dtype] * (parts[0][0].double().abs() + parts[1][0].double().abs())).all()
    assert (lse.double() - want_lse).abs().max() <= 3e-4


# --------------------------------------------------------------------- trim

def trimmed(t, named, window, sinks):
    table, lens, refs = (x.cpu().clone() for x in t)
    for s in {s for s in named if 0 <= s < table.shape[0]}:
        for c in range(-(-int(lens[s]) // 128)):
            if 128 * c >= sinks and 128 * (c + 1) <= int(lens[s]) - window + 1 and table[s, c] >= 0:
                refs[table[s, c]] -= 1
                table[s, c] = -1
    return table, lens, refs


@pytest.mark.parametrize("seqs,width,pages", [(8, 4, 40), (300, 9, 1500), (1200, 3, 3000), (5, 70, 9001)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (128, 0), (129, 130), (300, 128), (2 ** 31 - 1, 7), (50, 2 ** 31 - 300)])
def test_trim(paged, seqs, width, pages, window, sinks):
    t, data, cache = model_of(paged, seqs, width, pages, seqs + 2)
    old = [x.clone() for x in t]
    named = list(range(0, seqs, 2)) + [0, -1, seqs, 2]
    new = cache.trim(t, named, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip(t, old))
    for _ in range(2):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(new, trimmed(t, named, window, sinks)))
        new = cache.trim(new, named, window, sinks)   # what is gone is not given back twice
    given = paged.PageTables(*(torch.full_like(x, 55) for x in t))
    assert cache.trim(t, named, window, sinks, out=given) is given and all(torch.equal(a, b) for a, b in zip(given, new))
    assert all(torch.equal(a, b) for a, b in zip(cache.trim(t, [], window), t))


def test_new_tables_are_tensors_like_others(paged):
    """Whatever memory they share: written in place, saved, moved, made in inference mode and in a graph."""
    import io

    t, data, cache = model_of(paged, 8, 20, 200, 9)
    want = trimmed(t, [0, 2, 4, 6], 100, 3)
    for mode in (torch.inference_mode, torch.no_grad, torch.enable_grad):
        with mode():
            new = cache.trim(t, [0, 2, 4, 6], 100, 3)
            assert all(torch.equal(a.cpu(), b) and a.is_contiguous() for a, b in zip(new, want))
            new.lens.add_(1)
            new.refs.zero_()
            assert torch.equal(new.block_table.cpu(), want[0]) and torch.equal(new.lens.cpu(), want[1] + 1)
    file = io.BytesIO()
    torch.save(tuple(new), file)
    file.seek(0)
    assert all(torch.equal(a, b) for a, b in zip(torch.load(file), new))
    named, graph = ints([0, 2, 4, 6]), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        made = cache.trim(cache.trim(t, named, 100, 3), named, 100, 3)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(made, want))


def test_tables_after_a_trim(paged):
    """Trimmed sequences grow, fork, move and end like others."""
    t, data, cache = model_of(paged, 12, 40, 400, 3, share=False)
    window, sinks = 200, 4
    t = cache.trim(t, list(range(12)), window, sinks)
    table, lens, refs = (x.cpu() for x in t)
    assert (table[:, :1][lens[:, None] > 500] >= 0).all() and refs.sum() == (table >= 0).sum()
    alive = [s for s in range(12) if lens[s] > 0]
    t, granted = cache.reserve(t, alive, [min(40 * 128, int(lens[s]) + 100) for s in alive])
    assert granted.all()
    empty = [s for s in range(12) if lens[s] == 0]
    parent = max(alive, key=lambda s: int(lens[s]))
    t, granted = cache.fork(t, [parent] * len(empty), empty)
    assert granted.all()
    t, moved, live = cache.compact(t)
    table, lens, refs = (x.cpu() for x in t)
    used = refs > 0
    assert int(live) == int(used.sum()) and used[:int(live)].all() and refs.sum() == (table >= 0).sum()
    t = cache.free(t, list(range(12)))
    assert not t.refs.any() and (t.block_table == -1).all()


def test_attention_after_a_trim(paged):
    """A long stream, step by step: append, attend with sinks, trim; its rows are what they are without trimming."""
    heads, kv_heads, window, sinks, steps = 8, 2, 300, 5, 12
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = paged.CachePages([[torch.full((40, 128, kv_heads, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2)]])
    t = paged.PageTables(torch.full((2, 30), -1, dtype=torch.int32, device="cuda"), ints([0, 0]), ints([0] * 40))
    keys, values, most = [[], []], [[], []], 0
    for step in range(steps):
        new = [[700, 130, 1, 1, 77, 1, 400, 1, 200, 1, 3, 128][step], [90, 1, 1, 600, 1, 1, 1, 250, 1, 140, 1, 1][step]]
        lens = [int(x) + n for x, n in zip(t.lens, new)]
        t, granted = cache.reserve(t, [0, 1], lens)
        assert granted.tolist() == [1, 1]
        chunk = paged.Chunk(t.block_table, ints([0, new[0], sum(new)]), t.lens, max_q=max(new))
        q, k, v = (torch.randn((sum(new), h, 128), generator=g, device="cuda").bfloat16() for h in (heads, kv_heads, kv_heads))
        paged.append(cache.layers[0], chunk, None, k, v)
        out = paged.attend(cache.layers[0], chunk, q, window=window, sinks=sinks)
        for s in range(2):
            rows = slice(0, new[0]) if s == 0 else slice(new[0], sum(new))
            keys[s].append(k[rows])
            values[s].append(v[rows])
            kk, vv = (torch.cat(x).double().repeat_interleave(heads // kv_heads, 1) for x in (keys[s], values[s]))
            pos, key = torch.arange(lens[s] - new[s], lens[s], device="cuda")[:, None], torch.arange(lens[s], device="cuda")
            seen = (key <= pos) & ((key > pos - window) | (key < sinks))
            x = (torch.einsum("qhd,khd->hqk", q[rows].double(), kk) * 128 ** -0.5).masked_fill(~seen, -math.inf)
            w = torch.softmax(x, -1)
            want, mass = torch.einsum("hqk,khd->qhd", w, vv), torch.einsum("hqk,khd->qhd", w, vv.abs())
            assert ((out[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2e-4) * mass + 1e-7).all()
        t = cache.trim(t, [0, 1], window, sinks)
        # Freed pages hold nothing that is read again.
        free = (t.refs == 0).nonzero()[:, 0]
        for x in (cache.layers[0].k, cache.layers[0].v):
            x[free] = math.nan
        most = max(most, int((t.refs > 0).sum()))
    assert most <= 2 * (1 + 4) and int(t.lens.sum()) > 2500


@pytest.mark.parametrize("answers,prompt,dtype", [(2, 300, torch.bfloat16), (24, 2300, torch.float16), (40, 5000, torch.bfloat16)])
def test_answers_from_a_prompt_to_their_end(paged, answers, prompt, dtype):
    """Reserve, append, fork, and then token by token: append, find what is shared, attend with it, and the same from
    two parts joined.  All that the answers have in common is found, and every way gives one result."""
    heads, kv_heads, pages = 32, 8, 60 + 2 * answers
    g = torch.Generator(device="cuda").manual_seed(answers)
    cache = paged.CachePages([[torch.full((pages, 128, kv_heads, 128), math.nan, dtype=dtype, device="cuda") for _ in range(2)]])
    layer, rotary = cache.layers[0], paged.Rotary(base=500000.0, device="cuda:0")
    t = paged.PageTables(torch.full((answers, 50), -1, dtype=torch.int32, device="cuda"), ints([0] * answers), ints([0] * pages))
    t, granted = cache.reserve(t, [0], [prompt])
    assert granted.tolist() == [1]
    rand = lambda n, h: torch.randn((n, h, 128), generator=g, device="cuda").to(dtype)  # noqa: E731
    first = paged.Chunk(t.block_table[:1], ints([0, prompt]), t.lens[:1])
    paged.append(layer, first, None, rand(prompt, kv_heads), rand(prompt, kv_heads), rotary=rotary)
    t, granted = cache.fork(t, [0] * (answers - 1), list(range(1, answers)))
    assert granted.all()
    for step in range(3):
        t, granted = cache.reserve(t, list(range(answers)), [prompt + step + 1] * answers)
        assert granted.all()
        chunk = paged.Chunk(t.block_table, ints(list(range(answers + 1))), t.lens, max_q=1)
        q = paged.append(layer, chunk, 2 * rand(answers, heads), rand(answers, kv_heads), rand(answers, kv_heads), rotary=rotary)
        shared, common = paged.SharedPrefix(chunk), prompt // 128 * 128
        assert shared.tokens.tolist() == [common] * answers
        apart, apart_lse = paged.attend(layer, chunk, q, return_lse=True)
        out, lse = paged.attend(layer, chunk, q, shared=shared, return_lse=True)
        head = paged.Chunk(t.block_table, chunk.cu_q, ints([common] * answers), max_q=1)
        rest = paged.Chunk(t.block_table[:, common // 128:], chunk.cu_q, t.lens - common, max_q=1)
        parts = [paged.attend(layer, head, q, causal=False, return_lse=True), paged.attend(layer, rest, q, return_lse=True)]
        joined, joined_lse = paged.join(*zip(*parts))
        rows = t.block_table.long()
        k, v = (x[rows].flatten(1, 2)[:, :prompt + step + 1].double().repeat_interleave(heads // kv_heads, 2) for x in (layer.k, layer.v))
        x = torch.einsum("shd,skhd->shk", q.double(), k) * 128 ** -0.5
        w = torch.softmax(x, -1)
        want, mass = torch.einsum("shk,skhd->shd", w, v), torch.einsum("shk,skhd->shd", w, v.abs())
        tail = (prompt + 3) * 2.0 ** -25 * v.abs().amax() if dtype == torch.float16 else 0.0
        bound = EPS[dtype] * want.abs() + (EPS[dtype] + 2e-4) * mass + tail + 1e-7
        for got, got_lse in ((apart, apart_lse), (out, lse)):
            assert ((got.double() - want).abs() <= bound).all()
            assert (got_lse.double() - torch.logsumexp(x, -1)).abs().max() <= 3e-4
        # The parts were rounded once more.
        assert ((joined.double() - want).abs() <= bound + EPS[dtype] * sum(p[0].double().abs() for p in parts)).all()
        assert (joined_lse.double() - torch.logsumexp(x, -1)).abs().max() <= 3e-4
    t = cache.free(t, list(range(answers)))
    assert not t.refs.any()


# ----------------------------------------------------------------- refusals

def test_refusals(paged):
    c = Family(paged, [(1, 300), (1, 290)], [(2, 2)], 8, 2)
    other = paged.Chunk(c.chunk.block_table, c.chunk.cu_q, c.chunk.kv_lens)
    cache = paged.CachePages([[c.k, c.v]])
    t = paged.PageTables(c.chunk.block_table, c.chunk.kv_lens, torch.ones(cache.pages, dtype=torch.int32, device="cuda"))
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    attend = lambda **kw: paged.attend(c.pages, c.chunk, c.q, **kw)  # noqa: E731
    big = torch.zeros((4, 8, 128), dtype=c.dtype, device="cuda")
    bad = [
        lambda: attend(sinks=4),
        lambda: attend(window=8, sinks=-1),
        lambda: attend(window=8, sinks=1 << 31),
        lambda: attend(window=8, sinks=4, causal=False),
        lambda: attend(shared=c.shared, window=8),
        lambda: attend(shared=c.shared, window=8, sinks=2),
        lambda: paged.attend(c.pages, other, c.q, shared=c.shared),
        lambda: paged.SharedPrefix(c.chunk, ints([0])),
        lambda: paged.SharedPrefix(c.chunk, max_common=0),
        lambda: paged.SharedPrefix(c.chunk, ints([0, 1, 2, 2])),
        lambda: paged.SharedPrefix(c.chunk, torch.tensor([0, 2], device="cuda")),
        lambda: paged.SharedPrefix(c.chunk, torch.tensor([0, 2], dtype=torch.int32)),
        lambda: paged.join([out], [lse, lse]),
        lambda: paged.join([out] * 9, [lse] * 9),
        lambda: paged.join([out.float()], [lse]),
        lambda: paged.join([out, out.half()], [lse, lse]),
        lambda: paged.join([out, out[:1]], [lse, lse]),
        lambda: paged.join([out], [lse.double()]),
        lambda: paged.join([out], [lse[:1]]),
        lambda: paged.join([out], [lse.cpu()]),
        lambda: paged.join([out[..., :64]], [lse]),
        lambda: paged.join([out], [lse], out=out[:1]),
        lambda: paged.join([big[:2], big[2:]], [lse, lse], out=big[1:3]),
        lambda: paged.join([big[:2], big.transpose(0, 1)[:2, :, :].expand(2, 4, 128)], [lse, lse]),
        lambda: cache.trim(t, [0], 0),
        lambda: cache.trim(t, [0], 1 << 31),
        lambda: cache.trim(t, [0], 5, -1),
        lambda: cache.trim(t, torch.tensor([0], device="cuda"), 5),
        lambda: cache.trim(t, [0], 5, out=t),
        lambda: cache.trim(tuple(t), [0], 5),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    out, lse = c.run(paged)
    c.check(out, lse)
    assert paged.attend(c.pages, c.chunk, c.q[:0], shared=c.shared).shape == (0, 8, 128)
    assert paged.attend(c.pages, c.chunk, c.q[:0], window=3, sinks=1).shape == (0, 8, 128)


def test_offsets_past_two_gigabytes(paged):
    """Pages of a large cache, and partial results of many rows, need more than 32 bits."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 25 GB")
    pages = 20000
    k, v = (torch.zeros((pages, 128, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for lens in ([(1, 500), (130, 500), (2, 500)], [(1, 500), (4, 510), (2, 500)]):
        c = Family(paged, lens, [(3, 2)], 32, 8, spare=0)
        where = {p: q for p, q in zip(sorted(set(c.table[c.table >= 0].tolist())), range(pages - 1, 0, -1211))}
        table = c.chunk.block_table.clone()
        for p, q in where.items():
            k[q], v[q] = c.k[p], c.v[p]
            table[c.chunk.block_table == p] = q
        layer, chunk = paged.LayerPages(k, v), paged.Chunk(table, c.chunk.cu_q, c.chunk.kv_lens)
        whole = paged.SharedPrefix(chunk)
        assert together(layer, chunk, c.q, whole) == c.saves()
        c.check(paged.attend(layer, chunk, c.q, shared=whole))
        c.check(paged.attend(layer, chunk, c.q, window=100, sinks=3), window=100, sinks=3)
    assert c.saves()
    outs = [torch.full((70000, 128, 128), float(i), dtype=torch.bfloat16, device="cuda") for i in range(2)]
    lses = [torch.zeros((70000, 128), device="cuda") for _ in range(2)]
    outs[1][-1, -1] = 3.0
    out, lse = paged.join(outs, lses)
    assert (out[:-1] == 0.5).all() and (out[-1, -1] == 1.5).all() and (lse == lses[0] + math.log(2)).all()
