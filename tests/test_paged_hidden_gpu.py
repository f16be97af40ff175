"""Keys that no row sees between sinks and window, with each odd value in turn:
whole pages there have been given away, parts of a page beside what is seen hold
what they hold."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_paged_more_gpu import Seen  # noqa: E402


@pytest.fixture(scope="module")
def paged():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from secure_infer_b200 import paged
    return paged


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("lens", [[(1, 1000), (6, 1000), (150, 1000)], [(1, 130), (3, 200), (40, 250)], [(1, 20000)],
                                  [(300, 3000)]])
@pytest.mark.parametrize("window,sinks", [(100, 4), (60, 100), (200, 128), (33, 140), (1, 1)])
def test_hidden_keys_with_odd_values_change_no_bit(paged, lens, window, sinks, value):
    c = Seen(paged, lens, 8, 2)
    want, want_lse = c.attend(paged, window, sinks)
    c.check(want, want_lse, window=window, sinks=sinks)
    before = c.v.clone()
    gone = [c.hide(s, window, sinks, value) for s in range(len(lens))]
    changed = ~((c.v == before) | (torch.isnan(c.v) & torch.isnan(before)))
    # Keys between the sinks and the first row's window, of the lengths that have any.
    hidden = sum(max(0, max(0, kv - n - window + 1) - sinks) for n, kv in lens)
    assert changed.any(3).sum() == hidden * 2
    expected = torch.tensor(value).to(c.dtype).cuda()
    assert (torch.isnan(c.v[changed]) if math.isnan(value) else c.v[changed] == expected).all()
    assert [int((row < 0).sum()) - (c.table.shape[1] - -(-kv // 128)) for row, (_, kv) in zip(c.table, lens)] == gone
    c.chunk.block_table.copy_(c.table)
    out, lse = c.attend(paged, window, sinks)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
