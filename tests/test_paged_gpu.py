"""Operators on the paged cache against their definitions in 64 bits: attention
of a chunk, rotary append, and the page tables against a plain Python model.

Bounds.  An output of ``attend`` is rounded once (eps |o|), and each weight is
rounded once to the cache's type for the product with the values: eps times the
softmax of |v|.  Scores, exponentials and sums are 32-bit: 128 products of a
score lose at most 128 2^-24 of sum |q k|, below 2e-4 at these inputs, which is
a relative 2e-4 of every weight.  fp16 weights below 2^-14 round to multiples of
2^-24: up to 2^-25 |v| per key.  ``append`` rounds once, after angles that are
exact to 2^-24 of a turn."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# Unit roundoff: 8 and 11 significant bits.
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from secure_infer_b200 import paged
    return paged


class Case:
    """Random pages for sequences of (new, all) tokens; unwritten slots, unused
    pages and one page that no table names hold NaN."""

    def __init__(self, paged, lens, heads, kv_heads, dtype=torch.bfloat16, seed=0, layout="plain", spare=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.dtype, self.group = lens, dtype, heads // kv_heads
        used = [-(-kv // 128) for _, kv in lens]
        pages = sum(used) + spare
        order = torch.randperm(pages, generator=g, device="cuda").tolist()
        width = max(1, max(used)) + 2
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(used):
            table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        if layout == "heads":      # [pages, heads, 128, 128] seen as [pages, 128, heads, 128]
            kv = [torch.full((pages, kv_heads, 128, 128), math.nan, dtype=dtype, device="cuda").transpose(1, 2)
                  for _ in range(2)]
        elif layout == "joint":    # K and V of a page side by side
            both = torch.full((pages, 2, 128, kv_heads, 128), math.nan, dtype=dtype, device="cuda")
            kv = [both[:, 0], both[:, 1]]
        else:
            kv = [torch.full((pages, 128, kv_heads, 128), math.nan, dtype=dtype, device="cuda") for _ in range(2)]
        self.rows = []
        for s, (_, n) in enumerate(lens):
            k, v = (torch.randn((n, kv_heads, 128), generator=g, device="cuda", dtype=dtype) for _ in range(2))
            for c, x in zip(kv, (k, v)):
                for i in range(0, n, 128):
                    c[table[s, i // 128].item(), :min(128, n - i)] = x[i:i + 128]
            self.rows.append([k, v])
        self.k, self.v = kv
        self.cu = [0]
        for n, _ in lens:
            self.cu.append(self.cu[-1] + n)
        self.q = 2 * torch.randn((self.cu[-1], heads, 128), generator=g, device="cuda", dtype=dtype)
        self.table = table.cuda()
        self.pages = paged.LayerPages(self.k, self.v)
        self.chunk = paged.Chunk(self.table, torch.tensor(self.cu, dtype=torch.int32, device="cuda"),
                                 torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda"),
                                 max_q=max(n for n, _ in lens))

    def set_row(self, s, token, head, k=None, v=None):
        page, slot = self.table[s, token // 128].item(), token % 128
        for which, x in ((0, k), (1, v)):
            if x is not None:
                (self.k, self.v)[which][page, slot, head] = x
                self.rows[s][which][token, head] = x

    def expected(self, causal=True, window=0, scale=None):
        """(out, lse, bound) in 64 bits.  Hidden keys are left out, not weighted with zero."""
        scale = 128 ** -0.5 if scale is None else scale
        eps = EPS[self.dtype]
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        lse = torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        for s, (n, kv) in enumerate(self.lens):
            if n == 0 or kv == 0:
                continue
            k, v = (x.double().repeat_interleave(self.group, 1) for x in self.rows[s])
            x = torch.einsum("qhd,khd->hqk", self.q[self.cu[s]:self.cu[s + 1]].double(), k) * scale
            pos = torch.arange(kv - n, kv, device="cuda")[:, None]
            key = torch.arange(kv, device="cuda")[None]
            hidden = (key > pos) if causal else torch.zeros((n, kv), dtype=torch.bool, device="cuda")
            if window:
                hidden |= pos - key >= window
            x = x.masked_fill(hidden, -math.inf)
            some = ~hidden.all(1)
            w = torch.softmax(x, -1).masked_fill(hidden, 0.0)
            bad = ~torch.isfinite(v)
            o = torch.einsum("hqk,khd->qhd", w, v.masked_fill(bad, 0.0))
            # Visible infinities and NaN reach the rows that see them.
            if bad.any():
                seen = (~hidden).double()
                for value in (math.inf, -math.inf, math.nan):
                    at = torch.isnan(v) if math.isnan(value) else v == value
                    o = torch.where(torch.einsum("qk,khd->qhd", seen, at.double()) > 0, o + value, o)
            mass = torch.einsum("hqk,khd->qhd", w, v.abs().masked_fill(bad, 0.0))
            tail = kv * 2.0 ** -25 * v.abs().masked_fill(bad, 0.0).amax() if self.dtype == torch.float16 else 0.0
            rows = slice(self.cu[s], self.cu[s + 1])
            out[rows] = torch.where(some[:, None, None], o, 0.0)
            bound[rows] = eps * o.abs() + (eps + 2e-4) * mass + tail + 1e-7
            lse[rows] = torch.where(some[:, None], torch.logsumexp(x, -1).T, -math.inf)
        return out, lse, bound

    def check(self, got, lse=None, **kw):
        out, want_lse, bound = self.expected(**kw)
        got = got.double()
        fine = torch.isfinite(out)
        assert torch.equal(torch.isnan(got), torch.isnan(out))
        assert torch.equal(got[~fine & ~torch.isnan(out)], out[~fine & ~torch.isnan(out)])
        over = ((got - out).abs() - bound)[fine]
        assert over.numel() == 0 or over.max() <= 0, f"off by {over.max().item()} over the bound"
        if lse is not None:
            assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
            some = ~torch.isinf(want_lse)
            assert not some.any() or (lse.double() - want_lse)[some].abs().max() <= 3e-4


EDGES = [1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 255, 256, 257, 640, 1000]


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (8, 1), (4, 4), (7, 1), (40, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens_at_page_edges(paged, heads, kv_heads, dtype):
    c = Case(paged, [(1, n) for n in EDGES], heads, kv_heads, dtype)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("n", [2, 3, 5, 8, 13, 16, 17])
@pytest.mark.parametrize("heads,kv_heads", [(16, 4), (7, 1)])
def test_drafts(paged, n, heads, kv_heads):
    c = Case(paged, [(n, n), (n, 128), (n, 129 + n), (n, 700)], heads, kv_heads, seed=n)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (28, 4), (3, 3), (160, 1)])
@pytest.mark.parametrize("lens", [[(100, 100)], [(129, 300)], [(257, 1500)], [(64, 128), (0, 50), (200, 1000), (1, 900)],
                                  [(511, 640), (33, 33)]])
def test_chunks(paged, heads, kv_heads, lens):
    c = Case(paged, lens, heads, kv_heads, seed=len(lens))
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 500])
@pytest.mark.parametrize("lens", [[(1, n) for n in (1, 100, 128, 129, 777)], [(5, 700), (5, 5)], [(200, 900), (70, 70)]])
def test_window(paged, window, lens):
    c = Case(paged, lens, 8, 2, seed=window)
    out, lse = paged.attend(c.pages, c.chunk, c.q, window=window, return_lse=True)
    c.check(out, lse, window=window)


@pytest.mark.parametrize("lens", [[(1, 300)], [(9, 300), (4, 4)], [(150, 400), (150, 150)]])
def test_every_key(paged, lens):
    c = Case(paged, lens, 8, 2)
    out, lse = paged.attend(c.pages, c.chunk, c.q, causal=False, return_lse=True)
    c.check(out, lse, causal=False)


@pytest.mark.parametrize("lens", [[(0, 0), (1, 40), (0, 300), (1, 128), (0, 0)], [(3, 0), (1, 0)], [(1, 0), (200, 0), (130, 50)]])
def test_empty_sequences_and_rows(paged, lens):
    """Slots without new tokens, sequences without tokens, and more new tokens than the sequence holds: the rows
    before its first token see nothing."""
    c = Case(paged, lens, 8, 2)
    out = torch.full_like(c.q, math.nan)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True, out=out)
    c.check(out, lse)


@pytest.mark.parametrize("lens", [[(4, 200)], [(16, 130)], [(140, 400)], [(300, 300)]])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_that_later_tokens_hold_do_not_leak(paged, lens, value):
    """A row is what it is whatever the keys after it hold; rows that see the value get it."""
    c = Case(paged, lens, 8, 2, seed=3)
    n, kv = lens[0]
    c.set_row(0, kv - n // 2, 1, k=1.0, v=value)
    c.set_row(0, kv - 2, 0, k=value if not math.isinf(value) else 7.0)
    out = paged.attend(c.pages, c.chunk, c.q)
    first = n - 2
    got, (want, _, bound) = out.double(), c.expected()
    # Rows before any such key, and after it for the value (the key's NaN makes whole rows of head 0's group NaN).
    h = c.group
    assert torch.isfinite(got[:first, :h]).all()
    assert ((got - want).abs() <= bound)[:first, :h].all()
    if math.isnan(value):
        assert torch.isnan(got[first:, :h]).all()
    before, after = got[:n - n // 2, h:], got[n - n // 2:, h:]
    assert ((before - want[:n - n // 2, h:]).abs() <= bound[:n - n // 2, h:]).all()
    assert torch.isnan(after).all() if math.isnan(value) else torch.equal(after, torch.full_like(after, value))


def test_keys_left_of_a_window_may_hold_anything(paged):
    """Pages before a sliding window may have been given away: their table entries are stale."""
    c = Case(paged, [(1, 1000), (6, 1000), (150, 1000)], 8, 2)
    want = paged.attend(c.pages, c.chunk, c.q, window=200)
    c.check(want, window=200)
    for s, first in ((0, 800), (1, 795), (2, 651)):
        for p in range(first // 128):
            page = c.table[s, p].item()
            c.k[page] = math.nan
            c.v[page] = math.nan
        for x in (c.k, c.v):
            x[c.table[s, first // 128].item(), :first % 128] = math.nan
        c.table[s, :first // 128] = -7
    assert torch.equal(paged.attend(c.pages, c.chunk, c.q, window=200), want)


@pytest.mark.parametrize("layout", ["heads", "joint"])
@pytest.mark.parametrize("lens", [[(1, 300), (1, 77)], [(3, 300)], [(150, 500)]])
def test_layouts_and_strides(paged, layout, lens):
    c = Case(paged, lens, 12, 2, layout=layout)
    qkv = torch.randn((c.q.shape[0], 12 + 4, 128), device="cuda").to(c.dtype)
    qkv[:, 2:14] = c.q
    table = torch.full((len(lens), c.table.shape[1] + 5), 99, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    chunk = paged.Chunk(table[:, :c.table.shape[1]], c.chunk.cu_q, c.chunk.kv_lens)
    c.check(paged.attend(c.pages, chunk, qkv[:, 2:14]))


def test_scale(paged):
    c = Case(paged, [(1, 300), (40, 200)], 8, 2)
    for scale in (0.3, -0.05, 0.0):
        c.check(paged.attend(c.pages, c.chunk, c.q, scale=scale), scale=scale)


def test_large_scores(paged):
    """Scores of some thousands: only the running maximum keeps the exponentials in range."""
    c = Case(paged, [(1, 1000), (100, 700)], 4, 1)
    c.q.mul_(64)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    want, want_lse, _ = c.expected()
    assert torch.isfinite(out).all()
    # The scores' own 32-bit error grows with them: 128 2^-24 sum |q k| scale is below 0.02 here.
    assert (lse.double() - want_lse).abs().max() <= 2e-2
    assert (out.double() - want).abs().max() <= 0.05 * want.abs().max()


@pytest.mark.parametrize("lens,heads,kv_heads", [([(1, 20000)], 8, 1), ([(1, 5000), (1, 10)], 8, 8), ([(7, 9000)], 8, 1),
                                                 ([(100, 9000)], 8, 1), ([(1, 3), (300, 6000), (1, 2222)], 16, 2)])
def test_split_contexts_and_their_repetition(paged, lens, heads, kv_heads):
    """One long context is cut over many CTAs; repeated calls give the same bits whatever CTA finishes last."""
    c = Case(paged, lens, heads, kv_heads)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    c.check(out, lse)
    for _ in range(20):
        again, again_lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("lens", [[(1300, 1300)], [(3, 40), (700, 2000), (1, 300), (1100, 1100)]])
@pytest.mark.parametrize("window", [0, 150])
def test_sequences_of_many_tiles(paged, lens, window):
    """More tiles of a sequence than a warp has lanes, before and after others."""
    c = Case(paged, lens, 16, 1)
    out, lse = paged.attend(c.pages, c.chunk, c.q, window=window, return_lse=True)
    c.check(out, lse, window=window)


@pytest.mark.parametrize("lens", [[(300, 900)] + [(1, 3000)] * 20, [(1, 20000), (40, 50)], [(1, 5), (600, 4000), (2, 1)],
                                  [(40 if i % 7 == 0 else 1, 40 + (i * 37) % 300) for i in range(700)]])
def test_chunks_beside_single_tokens(paged, lens):
    """Both kinds share the SMs, whichever has more work; repeated calls give the same bits."""
    c = Case(paged, lens, 8, 2)
    out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
    c.check(out, lse)
    for _ in range(5):
        again, again_lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, again_lse)


def test_many_sequences(paged):
    """More sequences than a block has threads."""
    c = Case(paged, [(i % 4 != 3, 1 + (i * 37) % 300) for i in range(1500)], 4, 2)
    c.lens = [(int(n), kv) for n, kv in c.lens]
    c.check(paged.attend(c.pages, c.chunk, c.q))


def test_joining_two_halves(paged):
    """The statistics join attention over two sets of keys to attention over both."""
    c = Case(paged, [(1, 512)], 8, 2)
    whole, whole_lse = paged.attend(c.pages, c.chunk, c.q, causal=False, return_lse=True)
    parts = []
    for a, b in ((0, 2), (2, 4)):
        chunk = paged.Chunk(c.table[:, a:b].contiguous(), c.chunk.cu_q,
                            torch.tensor([256], dtype=torch.int32, device="cuda"), max_q=1)
        parts.append(paged.attend(c.pages, chunk, c.q, causal=False, return_lse=True))
    lse = torch.logaddexp(parts[0][1], parts[1][1])
    out = sum(o.float() * torch.exp(l - lse)[..., None] for o, l in parts)
    assert (lse - whole_lse).abs().max() <= 1e-5
    assert (out - whole.float()).abs().max() <= 2 ** -7 * whole.float().abs().max()


@pytest.mark.parametrize("lens", [[(1, 300), (1, 2000)], [(6, 900)], [(200, 1200), (1, 50)]])
def test_other_streams_and_graphs(paged, lens):
    c = Case(paged, lens, 8, 2)
    want = paged.attend(c.pages, c.chunk, c.q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = paged.attend(c.pages, c.chunk, c.q)
    side.synchronize()
    assert torch.equal(got, want)
    workspace, out = paged.attend_workspace("cuda:0"), torch.empty_like(c.q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(c.pages, c.chunk, c.q, out=out, workspace=workspace)
    # Same shapes, other contents.
    c.chunk.kv_lens.sub_(1)
    c.lens = [(n, kv - 1) for n, kv in c.lens]
    for s, (_, kv) in enumerate(c.lens):
        c.rows[s] = [x[:kv] for x in c.rows[s]]
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    c.check(out)


def test_pages_past_two_gigabytes(paged):
    """Offsets of a large cache need more than 32 bits."""
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 20 GB")
    pages = 20000
    k, v = (torch.zeros((pages, 128, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c = Case(paged, [(1, 256), (130, 256), (2, 256)], 32, 8, spare=0)
    table = c.table.clone()
    table[:, :2] = torch.tensor([[19999, 17000], [16384, 19998], [3, 16383]], dtype=torch.int32)
    for s in range(3):
        for i in range(2):
            k[table[s, i]], v[table[s, i]] = c.k[c.table[s, i]], c.v[c.table[s, i]]
    layer, chunk = paged.LayerPages(k, v), paged.Chunk(table, c.chunk.cu_q, c.chunk.kv_lens)
    c.check(paged.attend(layer, chunk, c.q))
    new = torch.randn((133, 8, 128), device="cuda").to(torch.bfloat16)
    paged.append(layer, chunk, None, new, new)
    assert torch.equal(k[17000, 127], new[0]) and torch.equal(v[19998, 127], new[130])
    whole = paged.CachePages([[k, v]])
    whole.copy([19998], [9])
    assert torch.equal(k[9], k[19998]) and torch.equal(v[9], v[19998])


# ------------------------------------------------------------------- append

def turned(x, positions, sections, base, interleaved):
    """x [tokens, heads, 128] in 64 bits."""
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    freq = torch.exp(-torch.arange(64, dtype=torch.float64) / 64 * math.log(base)).cuda()
    angle = positions.double()[axis].T * freq
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    x = x.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :64], x[..., 64:])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)


def near(got, want, dtype):
    # One rounding to the type, and 1e-6 of each term of the turn.
    return (got.double() - want).abs() <= EPS[dtype] * want.abs() + 2e-5


@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 200), (0, 0), (1, 129), (1, 128)], [(300, 300), (5, 900), (0, 40)]])
@pytest.mark.parametrize("sections,interleaved", [((64,), False), ((64,), True), ((16, 24, 24), False), ((0, 40, 24), True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append(paged, lens, sections, interleaved, dtype):
    c = Case(paged, lens, 12, 2, dtype)
    tokens = c.cu[-1]
    qkv = torch.randn((tokens, 16, 128), device="cuda").to(dtype)
    q, k, v = qkv[:, :12], qkv[:, 12:14], qkv[:, 14:]
    rotary = paged.Rotary(base=500000.0, sections=sections, interleaved=interleaved, device="cuda:0")
    positions = torch.randint(0, 1 << 20, (len(sections), tokens), dtype=torch.int32, device="cuda")
    before = [c.k.clone(), c.v.clone()]
    out = paged.append(c.pages, c.chunk, q, k, v, rotary=rotary, positions=positions)
    assert near(out, turned(q, positions, sections, 500000.0, interleaved), dtype).all()
    want_k = turned(k, positions, sections, 500000.0, interleaved)
    touched = torch.zeros(c.k.shape[:2], dtype=torch.bool, device="cuda")
    for s, (n, kv) in enumerate(lens):
        for i in range(n):
            page, slot, t = c.table[s, (kv - n + i) // 128].item(), (kv - n + i) % 128, c.cu[s] + i
            touched[page, slot] = True
            assert near(c.k[page, slot], want_k[t], dtype).all()
            assert torch.equal(c.v[page, slot], v[t])
    for now, old in ((c.k, before[0]), (c.v, before[1])):
        assert torch.equal(now[~touched].view(torch.int16), old[~touched].view(torch.int16))


def test_append_default_positions_and_plain_copy(paged):
    c = Case(paged, [(3, 130), (1, 1)], 4, 2)
    k, v = (torch.randn((4, 2, 128), device="cuda").to(c.dtype) for _ in range(2))
    assert paged.append(c.pages, c.chunk, None, k, v) is None
    assert torch.equal(c.k[c.table[0, 0], 127], k[0]) and torch.equal(c.k[c.table[0, 1], 1], k[2])
    rotary = paged.Rotary(device="cuda:0")
    q = torch.randn((4, 4, 128), device="cuda").to(c.dtype)
    out = paged.append(c.pages, c.chunk, q, k, v, rotary=rotary)
    places = torch.tensor([[127, 128, 129, 0]], device="cuda")
    assert near(out, turned(q, places, (64,), 10000.0, False), c.dtype).all()
    same = paged.append(c.pages, c.chunk, q, k, v, rotary=rotary, positions=places[0].int(), out=torch.empty_like(q))
    assert torch.equal(same, out)


def test_append_leaves_what_has_no_place(paged):
    """Entries outside the cache, places outside the table, tokens of nobody: queries turn, nothing is written."""
    c = Case(paged, [(4, 300), (2, 10)], 4, 2)
    c.table[0, 2] = 10 ** 6
    c.table[1, 0] = -1
    before = c.k.clone()
    k, v = (torch.randn((9, 2, 128), device="cuda").to(c.dtype) for _ in range(2))
    q = torch.randn((9, 4, 128), device="cuda").to(c.dtype)
    out = paged.append(c.pages, c.chunk, q, k, v)
    assert torch.equal(out, q) and torch.equal(c.k.view(torch.int16), before.view(torch.int16))
    chunk = paged.Chunk(c.table, c.chunk.cu_q, torch.tensor([2, 5000], dtype=torch.int32, device="cuda"))
    paged.append(c.pages, chunk, q, k, v)
    page = c.table[0, 0].item()
    assert torch.equal(c.k[page, 0], k[2]) and torch.equal(c.k[page, 1], k[3])
    before[page, :2] = k[2:4]
    assert torch.equal(c.k.view(torch.int16), before.view(torch.int16))


def test_rotary_keeps_its_precision_far_out(paged):
    """At position 2^30 a 32-bit product of position and frequency would be off by whole turns."""
    c = Case(paged, [(1, 1)], 2, 2)
    q = torch.randn((1, 2, 128), device="cuda").to(c.dtype)
    positions = torch.tensor([[(1 << 30) + 12345]], dtype=torch.int32, device="cuda")
    out = paged.append(c.pages, c.chunk, q, q, q, rotary=paged.Rotary(device="cuda:0"), positions=positions)
    assert near(out, turned(q, positions, (64,), 10000.0, False), c.dtype).all()


# ------------------------------------------------------------------- tables

def model_of(paged, seqs, width, pages, seed, share=True):
    """Random tables and the cache of three layers behind them."""
    r = torch.Generator().manual_seed(seed)
    table, lens, refs = torch.full((seqs, width), -1, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32), [0] * pages
    order, at = torch.randperm(pages, generator=r).tolist(), 0
    for s in range(seqs):
        if s % 3 == 2:
            continue
        n = int(torch.randint(0, width * 128 + 1, (1,), generator=r))
        used = -(-n // 128)
        if at + used > pages * 2 // 3:
            continue
        row = order[at:at + used]
        at += used
        if share and s and lens[0] >= 128 and used > 1:
            row[0] = int(table[0, 0])
            at -= 1
            order[at - len(row) + 1:at] = row[1:]
        for p in row:
            refs[p] += 1
        table[s, :used] = torch.tensor(row, dtype=torch.int32)
        lens[s] = n
    data = torch.randint(-30000, 30000, (3, 2, pages, 128, 1, 128), dtype=torch.int16, device="cuda").view(torch.bfloat16)
    tables = paged.PageTables(table.cuda(), lens.cuda(), torch.tensor(refs, dtype=torch.int32, device="cuda"))
    return tables, data, paged.CachePages([[d[0], d[1]] for d in data])


def bits(x):
    return x.view(torch.int16)


def consistent(t, extra=None):
    """Every used entry is a page, and each page's count is the rows that hold it."""
    table, lens, refs = (x.cpu() for x in t)
    counts = torch.zeros_like(refs)
    for row, n in zip(table, lens.tolist()):
        used = -(-n // 128)
        assert (row[:used] >= 0).all()
        for p in row[:used].tolist():
            counts[p] += 1
    return torch.equal(counts, refs)


@pytest.mark.parametrize("seqs,width,pages", [(8, 4, 40), (100, 9, 500), (1200, 3, 3000), (5, 70, 9001)])
def test_fork(paged, seqs, width, pages):
    t, data, cache = model_of(paged, seqs, width, pages, seqs)
    old = [x.clone() for x in t]
    image = data.clone()
    lens = t.lens.tolist()
    empty, full = [s for s in range(seqs) if lens[s] == 0], [s for s in range(seqs) if lens[s]]
    pairs = [(full[i % len(full)], e) for i, e in enumerate(empty)]
    pairs[1:1] = [(full[0], full[-1]), (full[0], empty[0]), (-1, empty[-1]), (full[0], seqs), (seqs, empty[-1])]
    new, granted = cache.fork(t, [p for p, _ in pairs], [c for _, c in pairs])
    assert all(torch.equal(a, b) for a, b in zip(t, old))
    free = [p for p in range(pages) if old[2][p] == 0]
    table, now, refs = old[0].cpu().clone(), old[1].cpu().clone(), old[2].cpu().clone()
    want, taken, seen, asked = [], [], set(), 0
    for parent, child in pairs:
        ok = 0 <= parent < seqs and 0 <= child < seqs and child not in seen and lens[child] == 0
        if 0 <= child < seqs:
            seen.add(child)
        need = int(ok and lens[parent] % 128 != 0)
        ok = ok and (not need or asked + need <= len(free))
        asked += need
        want.append(int(ok))
        if ok:
            k = lens[parent] // 128
            table[child] = -1
            table[child, :k] = old[0][parent, :k].cpu()
            for p in table[child, :k].tolist():
                refs[p] += 1
            if need:
                table[child, k] = free[asked - 1]
                refs[free[asked - 1]] += 1
                taken.append((int(old[0][parent, k]), free[asked - 1]))
            now[child] = lens[parent]
    assert granted.tolist() == want
    assert torch.equal(new.block_table.cpu(), table) and torch.equal(new.lens.cpu(), now) and torch.equal(new.refs.cpu(), refs)
    assert consistent(new)
    for src, dst in taken:
        image[:, :, dst] = image[:, :, src]
    assert torch.equal(bits(data), bits(image))


def test_fork_until_pages_run_out(paged):
    t, data, cache = model_of(paged, 12, 6, 30, 1, share=False)
    lens = t.lens.tolist()
    parent = next(s for s in range(12) if lens[s] % 128)
    refs = torch.ones_like(t.refs)
    refs[[7, 21]] = 0
    tight = paged.PageTables(t.block_table, t.lens, refs)
    children = [s for s in range(12) if lens[s] == 0]
    assert len(children) >= 4
    new, granted = cache.fork(tight, [parent] * len(children), children)
    assert granted.tolist() == [1, 1] + [0] * (len(children) - 2)
    k = lens[parent] // 128
    assert new.block_table[children[0], k] == 7 and new.block_table[children[1], k] == 21
    assert (new.lens[children[2:]] == 0).all()


@pytest.mark.parametrize("seqs,width,pages", [(8, 4, 40), (300, 9, 1500), (1200, 3, 3000)])
def test_reserve(paged, seqs, width, pages):
    t, data, cache = model_of(paged, seqs, width, pages, seqs + 1)
    old = [x.cpu().clone() for x in t]
    lens = old[1].tolist()
    r = torch.Generator().manual_seed(5)
    asks = [(s, min(width * 128, lens[s] + int(torch.randint(0, 300, (1,), generator=r)))) for s in range(seqs)]
    asks[2:2] = [(0, lens[0] - 1 if lens[0] else 1), (1, width * 128 + 1), (-1, 5), (seqs, 5)]
    new, granted = cache.reserve(t, [s for s, _ in asks], [n for _, n in asks])
    free = [p for p in range(pages) if old[2][p] == 0]
    table, now, refs, asked, seen = old[0].clone(), old[1].clone(), old[2].clone(), 0, set()
    want = []
    for s, n in asks:
        ok = 0 <= s < seqs and s not in seen
        seen.add(s)
        ok = ok and lens[s] <= n <= width * 128
        if ok and n > lens[s] and lens[s] % 128:
            ok = old[2][old[0][s, lens[s] // 128]] == 1
        need = -(-n // 128) - -(-lens[s] // 128) if ok else 0
        ok = ok and (need == 0 or asked + need <= len(free))
        if ok:
            table[s, -(-lens[s] // 128):-(-n // 128)] = torch.tensor(free[asked:asked + need], dtype=torch.int32)
            refs[free[asked:asked + need]] = 1
            now[s] = n
        asked += need
        want.append(int(ok))
    assert granted.tolist() == want and 0 < sum(want) < len(want)
    assert torch.equal(new.block_table.cpu(), table) and torch.equal(new.lens.cpu(), now) and torch.equal(new.refs.cpu(), refs)
    assert consistent(new)


@pytest.mark.parametrize("seqs,width,pages", [(8, 4, 40), (300, 9, 1500), (1200, 3, 3000)])
def test_free(paged, seqs, width, pages):
    t, data, cache = model_of(paged, seqs, width, pages, seqs + 2)
    old = [x.cpu().clone() for x in t]
    ended = list(range(0, seqs, 2)) + [0, -1, seqs, 2]
    new = cache.free(t, ended)
    table, lens, refs = (x.clone() for x in old)
    for s in range(0, seqs, 2):
        for p in table[s, :-(-int(lens[s]) // 128)].tolist():
            refs[p] -= 1
        table[s], lens[s] = -1, 0
    assert torch.equal(new.block_table.cpu(), table) and torch.equal(new.lens.cpu(), lens) and torch.equal(new.refs.cpu(), refs)
    assert consistent(new)
    assert torch.equal(cache.free(t, []).block_table, t.block_table)


@pytest.mark.parametrize("seqs,width,pages", [(8, 4, 40), (100, 9, 500), (1200, 3, 3000), (5, 70, 9001), (1, 1, 1)])
def test_compact(paged, seqs, width, pages):
    t, data, cache = model_of(paged, seqs, width, pages, seqs + 3)
    old = [x.cpu().clone() for x in t]
    image = data.clone()
    new, moved, live = cache.compact(t)
    used = [p for p in range(pages) if old[2][p] > 0]
    n = len(used)
    sources, holes = [p for p in used if p >= n], [p for p in range(n) if old[2][p] == 0]
    where = {p: p for p in used} | dict(zip(sources, holes))
    assert live.tolist() == [n] and moved.tolist() == [where.get(p, -1) for p in range(pages)]
    refs = torch.zeros_like(old[2])
    for p, q in where.items():
        refs[q] = old[2][p]
    assert torch.equal(new.refs.cpu(), refs) and torch.equal(new.lens.cpu(), old[1]) and consistent(new)
    for s in range(seqs):
        k = -(-int(old[1][s]) // 128)
        assert new.block_table[s, :k].tolist() == [where[p] for p in old[0][s, :k].tolist()]
        assert (new.block_table[s, k:] == -1).all()
    for src, dst in zip(sources, holes):
        image[:, :, dst] = image[:, :, src]
    assert torch.equal(bits(data), bits(image))


def test_copy_and_layouts(paged):
    data = torch.randint(-30000, 30000, (130, 20, 2, 128, 2, 128), dtype=torch.int16, device="cuda").view(torch.bfloat16)
    cache = paged.CachePages([[d[:, 0], d[:, 1].view(20, 2, 128, 128).transpose(1, 2)] for d in data])   # 260 tensors
    image = data.clone()
    cache.copy([3, 19, 0], [4, 2, 7])
    image[:, [4, 2, 7]] = image[:, [3, 19, 0]]
    assert torch.equal(bits(data), bits(image))
    cache.copy(torch.tensor([-1, 20, 5], dtype=torch.int32, device="cuda"), torch.tensor([1, 1, 99], dtype=torch.int32, device="cuda"))
    cache.copy([], [])
    assert torch.equal(bits(data), bits(image))


# ----------------------------------------------------------------- refusals

def test_refusals(paged):
    c = Case(paged, [(1, 300), (2, 20)], 8, 2)
    q = c.q
    bad = [
        lambda: paged.attend(c.pages, c.chunk, q[:, :7]),
        lambda: paged.attend(c.pages, c.chunk, q[..., :64]),
        lambda: paged.attend(c.pages, c.chunk, q.half()),
        lambda: paged.attend(c.pages, c.chunk, q.cpu()),
        lambda: paged.attend(c.pages, c.chunk, torch.empty((3, 8, 132), dtype=c.dtype, device="cuda")[..., 2:130]),
        lambda: paged.attend(c.pages, c.chunk, q, window=-1),
        lambda: paged.attend(c.pages, c.chunk, q, window=5, causal=False),
        lambda: paged.attend(c.pages, c.chunk, q, out=torch.empty_like(q)[:2]),
        lambda: paged.attend(c.pages, c.chunk, q, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")),
        lambda: paged.LayerPages(c.k, c.v[:-1]),
        lambda: paged.LayerPages(c.k[:, :64], c.v[:, :64]),
        lambda: paged.LayerPages(c.k.float(), c.v.float()),
        lambda: paged.LayerPages(c.k.cpu(), c.v.cpu()),
        lambda: paged.Chunk(c.table.long(), c.chunk.cu_q, c.chunk.kv_lens),
        lambda: paged.Chunk(c.table, c.chunk.cu_q[:-1], c.chunk.kv_lens),
        lambda: paged.Chunk(c.table, c.chunk.cu_q, c.chunk.kv_lens.cpu()),
        lambda: paged.Chunk(c.table, c.chunk.cu_q, c.chunk.kv_lens, max_q=-1),
        lambda: paged.append(c.pages, c.chunk, q, q, q),
        lambda: paged.append(c.pages, c.chunk, q, q[:, :2], q[:2, :2]),
        lambda: paged.append(c.pages, c.chunk, None, q[:, :2], q[:, :2], out=q),
        lambda: paged.append(c.pages, c.chunk, q, q[:, :2], q[:, :2], positions=c.chunk.kv_lens),
        lambda: paged.append(c.pages, c.chunk, q, q[:, :2], q[:, :2], rotary=paged.Rotary(sections=(32, 32), device="cuda:0"),
                             positions=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: paged.Rotary(sections=(10, 20), device="cuda:0"),
        lambda: paged.Rotary(base=0.0, device="cuda:0"),
        lambda: paged.CachePages([]),
        lambda: paged.CachePages([[c.k, c.v], [c.k[:-1], c.v[:-1]]]),
    ]
    cache = paged.CachePages([[c.k, c.v]])
    t = paged.PageTables(c.table.contiguous(), c.chunk.kv_lens, torch.ones(cache.pages, dtype=torch.int32, device="cuda"))
    bad += [
        lambda: cache.copy([1], [1]),
        lambda: cache.copy([1, 2], [3, 3]),
        lambda: cache.copy([1], [2, 3]),
        lambda: cache.copy([1], [cache.pages]),
        lambda: cache.free(t, torch.tensor([0], device="cuda")),
        lambda: cache.free(t._replace(refs=t.refs[:-1]), [0]),
        lambda: cache.free(t, [0], out=t),
        lambda: cache.free(tuple(t), [0]),
        lambda: cache.fork(t, [0], [1, 2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    # Nothing of it ran, and the operators still work.
    c.check(paged.attend(c.pages, c.chunk, c.q))
    empty = paged.attend(c.pages, c.chunk, q[:0])
    assert empty.shape == (0, 8, 128)


def test_given_tables(paged):
    """Tables to write into: refused where they overlap, else the same as new ones."""
    c = Case(paged, [(1, 300), (1, 77)], 8, 2)
    cache = paged.CachePages([[c.k, c.v]])
    refs = torch.zeros(cache.pages, dtype=torch.int32, device="cuda")
    refs[c.table[c.table >= 0].long()] = 1
    t = paged.PageTables(c.table.contiguous(), c.chunk.kv_lens, refs)
    fresh = lambda: paged.PageTables(*(torch.full_like(x, 55) for x in t))  # noqa: E731
    small = torch.empty(max(2, cache.pages), dtype=torch.int32, device="cuda")
    for out in (paged.PageTables(fresh().block_table, t.lens, fresh().refs), fresh()._replace(lens=small[:2], refs=small[:cache.pages]),
                fresh()._replace(refs=refs[:-1]), fresh()._replace(block_table=fresh().block_table[:, 1:].contiguous()),
                tuple(fresh())[:2], 3):
        with pytest.raises(ValueError):
            cache.free(t, [0], out=out)
        with pytest.raises(ValueError):
            cache.reserve(t, [0], [301], out=out)
        with pytest.raises(ValueError):
            cache.fork(t, [0], [1], out=out)
        with pytest.raises(ValueError):
            cache.compact(t, out=out)
    for run in (lambda out: cache.free(t, [0], out=out), lambda out: cache.reserve(t, [1, 0], [200, 299], out=out)[0],
                lambda out: cache.fork(t, [0], [1], out=out)[0]):
        want, given = run(None), fresh()
        assert run(given) is given
        for a, b in zip(want, given):
            assert torch.equal(a, b)



# ------------------------------------------------- workspaces of captured calls

@pytest.mark.parametrize("lens", [[(1, 9000)], [(100, 9000)], [(1, 4000), (300, 6000), (7, 2222)]])
def test_graphs_beside_eager_calls(paged, lens):
    """A graph captured on a stream that has called attend before, replayed on another while the first goes on: the two
    cut their tiles over the same CTAs and must not count each other's pieces."""
    a, b = Case(paged, lens, 8, 1, seed=1), Case(paged, lens, 8, 1, seed=2)
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        want_a, want_b = (paged.attend(c.pages, c.chunk, c.q) for c in (a, b))
    first.synchronize()
    a.check(want_a)
    b.check(want_b)
    out = [torch.empty_like(b.q) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, o in zip(graphs, out):
        with torch.cuda.graph(graph, stream=first):
            for _ in range(3):
                paged.attend(b.pages, b.chunk, b.q, out=o)
    got = []
    for i in range(40):
        with torch.cuda.stream(second):
            graphs[i % 2].replay()
        with torch.cuda.stream(first):
            graphs[1 - i % 2].replay()
            got += [paged.attend(a.pages, a.chunk, a.q) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_a) for x in got)
    assert all(torch.equal(o, want_b) for o in out)


def test_calls_of_one_capture_share_a_workspace(paged):
    """One per capture and stream, in the graph's memory, and another for the next."""
    c = Case(paged, [(1, 300)], 8, 2)
    side, fork = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    used, eager = [], paged._workspace(0, side.cuda_stream)
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            paged.attend(c.pages, c.chunk, c.q)
            used.append(paged._workspace(0, side.cuda_stream))
            paged.attend(c.pages, c.chunk, c.q)
            assert paged._workspace(0, side.cuda_stream) is used[-1]
            fork.wait_stream(side)
            with torch.cuda.stream(fork):
                assert paged._workspace(0, fork.cuda_stream) is not used[-1]
            side.wait_stream(fork)
    assert used[0] is not used[1] and all(w is not eager for w in used)
    assert paged._workspace(0, side.cuda_stream) is eager


# ------------------------------------------------- a workspace that is down

@pytest.mark.parametrize("lens,heads,kv_heads", [([(1, 300), (3, 40)], 8, 2), ([(1, 20000)], 8, 1), ([(200, 500)], 28, 4),
                                                 ([(100, 9000)], 8, 1), ([(1, 3000), (300, 2000), (0, 5), (2, 700)], 16, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_workspace_that_is_down_gives_nan_until_its_status_is_read(paged, lens, heads, kv_heads, dtype):
    """The host writes the status that a wait leaves when it runs out (and counts that were left behind); no wait runs
    out here."""
    c = Case(paged, lens, heads, kv_heads, dtype)
    workspace = paged.attend_workspace("cuda:0")
    out, lse = torch.zeros_like(c.q), None
    state = workspace.view(torch.int32)
    state[0] = 1
    state[64:200] = 3
    for _ in range(2):
        out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True, out=out, workspace=workspace)
        assert torch.isnan(out).all() and torch.isnan(lse).all()
    assert paged.attend_status(workspace) == 1
    assert paged.attend_status(workspace) == 0 and not workspace[:4096].any()
    for _ in range(2):
        out, lse = paged.attend(c.pages, c.chunk, c.q, return_lse=True, workspace=workspace)
        c.check(out, lse)
    assert paged.attend_status(workspace) == 0 and not workspace[:4096].any()


def test_status_of_the_streams_own_workspace(paged):
    c = Case(paged, [(1, 300)], 8, 2)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert paged.attend_status() == 0
        paged.attend(c.pages, c.chunk, c.q)
        paged._workspaces[0, side.cuda_stream][0] = 1
        assert torch.isnan(paged.attend(c.pages, c.chunk, c.q)).all()
        assert paged.attend_status() == 1 and paged.attend_status() == 0
        c.check(paged.attend(c.pages, c.chunk, c.q))
    with pytest.raises(ValueError):
        paged.attend_status(torch.zeros(8192, dtype=torch.uint8))
    with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
        with pytest.raises(RuntimeError):
            paged.attend_status(paged._workspaces[0, side.cuda_stream])


@pytest.mark.parametrize("lens", [[(5, 30000)], [(150, 20000)]])
def test_values_that_do_not_leak_after_long_contexts(paged, lens):
    """Rows taken key by key over a long context, while the kernel's other warps wait for them."""
    c = Case(paged, lens, 8, 1, seed=4)
    n, kv = lens[0]
    c.set_row(0, kv - n // 2, 0, v=math.inf)
    workspace = paged.attend_workspace("cuda:0")
    c.check(paged.attend(c.pages, c.chunk, c.q, workspace=workspace))
    assert paged.attend_status(workspace) == 0


# ------------------------------------------- requests that find too few pages

def test_reserve_goes_on_after_a_request_that_does_not_fit(paged):
    """Five free pages: ten do not fit, the two that the next one asks for do, then three, then none is left."""
    data = torch.zeros((1, 2, 8, 128, 1, 128), dtype=torch.bfloat16, device="cuda")
    cache = paged.CachePages([[d[0], d[1]] for d in data])
    t = paged.PageTables(torch.full((6, 12), -1, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda"),
                         torch.tensor([0, 1, 0, 0, 1, 0, 1, 0], dtype=torch.int32, device="cuda"))
    new, granted = cache.reserve(t, [0, 1, 2, 3, 4, 5], [1280, 256, 513, 384, 1, 0])
    assert granted.tolist() == [0, 1, 0, 1, 0, 1]
    assert new.lens.tolist() == [0, 256, 0, 384, 0, 0]
    assert new.block_table[1, :3].tolist() == [0, 2, -1] and new.block_table[3, :4].tolist() == [3, 5, 7, -1]
    assert (new.block_table[[0, 2, 4, 5]] == -1).all() and new.refs.tolist() == [1] * 8


@pytest.mark.parametrize("seqs,width,pages", [(40, 8, 60), (700, 9, 900), (3000, 5, 2500), (2500, 40, 20000)])
def test_reserve_with_few_pages(paged, seqs, width, pages):
    """Every request that fits into what the ones before it left is granted, and no other."""
    t, data, cache = model_of(paged, seqs, width, pages, seqs + 4, share=False)
    table, lens, refs = (x.cpu().clone() for x in t)
    r = torch.Generator().manual_seed(seqs)
    order = torch.randperm(seqs, generator=r).tolist()
    asks = [(s, min(width * 128, int(lens[s]) + int(torch.randint(0, width * 128, (1,), generator=r)))) for s in order]
    asks[seqs // 2:seqs // 2] = [(order[0], width * 128), (-1, 3), (seqs, 3)]
    new, granted = cache.reserve(t, [s for s, _ in asks], [n for _, n in asks])
    free, want, seen = [p for p in range(pages) if refs[p] == 0], [], set()
    some_after_a_refusal = False
    for s, n in asks:
        ok = 0 <= s < seqs and s not in seen
        seen.add(s)
        if ok:
            a, b = -(-int(lens[s]) // 128), -(-n // 128)
            ok = b - a <= len(free)
            if ok and b > a:
                some_after_a_refusal |= 0 in want
                table[s, a:b] = torch.tensor(free[:b - a], dtype=torch.int32)
                refs[free[:b - a]] = 1
                del free[:b - a]
        if ok:
            lens[s] = n
        want.append(int(ok))
    assert some_after_a_refusal
    assert granted.tolist() == want
    assert torch.equal(new.block_table.cpu(), table) and torch.equal(new.lens.cpu(), lens) and torch.equal(new.refs.cpu(), refs)
    assert consistent(new)


@pytest.mark.parametrize("lens", [[(10, 4)], [(200, 50), (3, 1), (1, 300)], [(300, 120)]])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 100000])
def test_windows_that_hide_nothing(paged, lens, window):
    """The largest windows, with rows at positions before the sequence's first."""
    c = Case(paged, lens, 8, 2, seed=6)
    out, lse = paged.attend(c.pages, c.chunk, c.q, window=window, return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("lens", [[(1, 300)], [(5, 700)], [(40, 1000)], [(200, 1000)], [(500, 2000)]])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (64, 32)])
def test_rows_whose_scores_are_all_minus_infinity(paged, lens, heads, kv_heads):
    """A query that meets keys of minus infinity alone has no softmax: NaN, as 0 / 0 is, and not an average of values.
    Rows that see one finite score have all their weight there."""
    c = Case(paged, lens, heads, kv_heads, seed=7)
    n, kv = lens[0]
    c.q[:, :, 0] = 1.0                                    # so that a key's minus infinity is its score's
    c.rows[0][0][:, ::2, 0] = -math.inf
    for i in range(0, kv, 128):
        c.k[c.table[0, i // 128], :min(128, kv - i), ::2, 0] = -math.inf
    odd = torch.arange(heads, device="cuda") // 2 % 2 == 1
    out = paged.attend(c.pages, c.chunk, c.q)
    assert torch.isnan(out[:, ~odd]).all()
    want, _, bound = c.expected()
    assert ((out.double() - want).abs() <= bound)[:, odd].all()
    for h in range(0, kv_heads, 2):
        c.set_row(0, 200, h, k=0.0)                       # one finite score, on a page after the first
    out, seen = paged.attend(c.pages, c.chunk, c.q)[:, ~odd], torch.arange(kv - n, kv, device="cuda") >= 200
    assert torch.isnan(out[~seen]).all()
    assert torch.equal(out[seen], c.rows[0][1][200, ::2].repeat_interleave(2, 0).expand_as(out[seen]))


@pytest.mark.parametrize("lens,heads,kv_heads", [([(600, 3000)], 28, 4), ([(300, 2500), (100, 1500)], 40, 8)])
def test_results_do_not_depend_on_what_shared_memory_held(paged, lens, heads, kv_heads):
    """Groups that do not fill a tile's 128 rows: after calls that leave finite values or NaN in shared memory, the same
    bits."""
    c = Case(paged, lens, heads, kv_heads, seed=8)
    before = Case(paged, [(1, 700)] * 80, 16, 8)
    got = []
    for value in (0.5, math.nan, 2.0, math.nan):
        before.k.fill_(value)
        before.v.fill_(value)
        paged.attend(before.pages, before.chunk, before.q)
        got.append(paged.attend(c.pages, c.chunk, c.q))
    c.check(got[0])
    assert all(torch.equal(g, got[0]) for g in got)


@pytest.mark.parametrize("lens", [[(500, 2500)], [(100, 1500), (250, 2000)]])
def test_results_do_not_depend_on_tokens_of_nobody(paged, lens):
    """Queries past the chunk's last token, as a padded step has them."""
    c = Case(paged, lens, 32, 8, seed=9)
    got = []
    for value in (0.0, math.nan, 50.0):
        q = torch.cat((c.q, torch.full((64, 32, 128), value, dtype=c.dtype, device="cuda")))
        got.append(paged.attend(c.pages, c.chunk, q)[:c.cu[-1]])
    c.check(got[0])
    assert all(torch.equal(g, got[0]) for g in got)


def test_workspaces_are_of_the_devices_size_and_can_be_given_up(paged):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    workspace = paged.attend_workspace("cuda")
    assert workspace.device == torch.device("cuda", 0)
    assert 0 < workspace.nbytes - 4 * 2 * sms * (256 + 8) * 130 < 16384   # two partial results a CTA, counters and cuts
    c = Case(paged, [(1, 20000), (300, 5000)], 8, 1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        with torch.cuda.stream(side):
            out = paged.attend(c.pages, c.chunk, c.q)
        side.synchronize()
        c.check(out)
        assert (0, side.cuda_stream) in paged._workspaces
        paged.release_workspaces(side)
        assert (0, side.cuda_stream) not in paged._workspaces
    paged.attend(c.pages, c.chunk, c.q)
    paged.release_workspaces()
    assert not paged._workspaces and not paged._captured
    # Nothing is written past a workspace of the size that is asked for.
    n = workspace.nbytes
    guarded = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    guarded[:n].zero_()
    c.check(paged.attend(c.pages, c.chunk, c.q, workspace=guarded[:n]))
    assert (guarded[n:] == 0x5A).all()


@pytest.mark.parametrize("through", ["python", "c"])
def test_a_host_thread_may_begin_with_attend(paged, through):
    """A thread that has called nothing else of CUDA."""
    import threading
    from secure_infer_b200 import _native
    c = Case(paged, [(1, 900), (200, 600)], 8, 2)
    want = paged.attend(c.pages, c.chunk, c.q)
    out, workspace = torch.empty_like(c.q), paged.attend_workspace("cuda:0")
    chunk = _native.Chunk.from_buffer_copy(c.chunk._c)
    chunk.tokens = c.q.shape[0]
    torch.cuda.synchronize()
    got = []

    def work():
        if through == "python":
            got.append(paged.attend(c.pages, c.chunk, c.q, out=out, workspace=workspace) is not None)
        else:
            got.append(_native.lib().secure_infer_paged_attend(
                c.pages._address, _native.ct.addressof(chunk), c.q.data_ptr(), c.q.stride(0), c.q.stride(1), 8, out.data_ptr(),
                None, 128 ** -0.5, 1, 0, workspace.data_ptr(), None) == 0)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert got == [True] and torch.equal(out, want)


def test_host_threads_that_share_a_stream_and_a_workspace(paged):
    """Each call is up to three launches that hand the workspace on; two threads' calls do not come between."""
    import threading
    from secure_infer_b200 import _native
    cases = [Case(paged, lens, 8, 1, seed=i) for i, lens in enumerate(([(300, 4000), (1, 900), (2, 70)], [(200, 6000), (1, 2500)]))]
    workspace, stream = paged.attend_workspace("cuda:0"), torch.cuda.Stream()
    torch.cuda.synchronize()
    want = [paged.attend(c.pages, c.chunk, c.q) for c in cases]
    outs = [[torch.empty_like(c.q) for _ in range(60)] for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(c, outs):
        chunk = _native.Chunk.from_buffer_copy(c.chunk._c)
        chunk.tokens = c.q.shape[0]
        for o in outs:   # ctypes lets the other thread run during the call
            bad.append(_native.lib().secure_infer_paged_attend(
                c.pages._address, _native.ct.addressof(chunk), c.q.data_ptr(), c.q.stride(0), c.q.stride(1), 8, o.data_ptr(),
                None, 128 ** -0.5, 1, 0, workspace.data_ptr(), stream.cuda_stream))

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    stream.synchronize()
    assert bad == [0] * 120
    for w, got in zip(want, outs):
        assert all(torch.equal(o, w) for o in got)


def test_wide_tables(paged):
    """A table for a hundred million tokens costs nothing by itself; work beyond 32 bits is a refused argument."""
    c = Case(paged, [(2048, 2100)], 8, 8)
    want = paged.attend(c.pages, c.chunk, c.q)
    table = torch.full((1, 1 << 20), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    assert torch.equal(paged.attend(c.pages, paged.Chunk(table, c.chunk.cu_q, c.chunk.kv_lens), c.q), want)
    many = Case(paged, [(2048, 2048)], 64, 64)
    table = torch.full((1, 1 << 22), -1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="more work"):
        paged.attend(many.pages, paged.Chunk(table, many.chunk.cu_q, many.chunk.kv_lens), many.q)


def test_memory_that_runs_out_is_torchs_error(paged):
    """A caller that makes room and tries again catches torch.OutOfMemoryError."""
    c = Case(paged, [(300, 300)], 64, 1)
    k = torch.zeros((300, 1, 128), dtype=c.dtype, device="cuda")
    want = paged.attend(c.pages, c.chunk, c.q)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / total)
    try:
        kept = []
        with pytest.raises(torch.OutOfMemoryError):
            for _ in range(1000):
                kept.append(paged.attend(c.pages, c.chunk, c.q))
        with pytest.raises(torch.OutOfMemoryError):
            paged.append(c.pages, c.chunk, c.q, k, k)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(paged.attend(c.pages, c.chunk, c.q), want)
