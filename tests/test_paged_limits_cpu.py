"""Bounds of the paged operators that the host keeps before anything is launched,
where there is no GPU."""
from __future__ import annotations

import ctypes as ct
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from secure_infer_b200 import _native

A = 1 << 20   # an address that is never read


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def sizes(seqs, tokens, width, heads, max_q=0):
    pages = _native.Pages(A, A, (ct.c_int64 * 3)(131072, 1024, 128), (ct.c_int64 * 3)(131072, 1024, 128), 10, heads, 0, 0)
    return pages, _native.Chunk(A, A, A, width, width, seqs, tokens, max_q)


# 2^20 sequences of one token with 24 rows on each of 8 KV heads are three tiles of few rows for each.  A tile's units
# are its pages and its cost, summed in 32 bits: at 84 pages 2139095040 with a cost of 1, 2164260864 with 2.
MANY = 1 << 20


def test_work_with_sinks_is_bounded_by_what_its_kernels_count(lib):
    call = lib.secure_infer_attend_fits_window
    pages, chunk = sizes(MANY, MANY, 84, 8)
    p, c = ct.byref(pages), ct.byref(chunk)
    assert 3 * MANY * 8 * (84 + 1) < 2 ** 31 <= 3 * MANY * 8 * (84 + 2)
    assert lib.secure_infer_attend_fits(p, c, 192) and call(p, c, 192, 0, 0) and call(p, c, 192, 10000, 0)
    assert not call(p, c, 192, 10000, 4)
    # A window or sinks as long as the table leave the usual call.
    assert call(p, c, 192, 84 * 128, 4) and call(p, c, 192, 10, 84 * 128) and call(p, c, 192, 2 ** 31 - 1, 2 ** 31 - 1)
    chunk.table_width = chunk.table_stride = 83
    assert call(p, c, 192, 10000, 4)
    # The call itself refuses it, before it reads anything.
    chunk.table_width = chunk.table_stride = 84
    options = _native.AttendOptions(None, None, 0, 0, 4)
    assert lib.secure_infer_attend(p, c, A, 192 * 128, 128, 192, A, None, 1.0, 1, 10000, ct.byref(options), A, None) == -1
    assert not call(None, c, 192, 10000, 4) and not call(p, None, 192, 10000, 4) and not call(p, c, 191, 10000, 4)


@pytest.mark.parametrize("seqs,q,width,group,apart", [
    (MANY, 1, 84, 24, "rows"),           # three tiles of few rows a sequence: a cost of 2, not 1
    (1 << 17, 75, 609, 4, "tiles"),      # 300 rows a sequence and again those of the prefix: a cost of 4, not 2
])
def test_work_with_a_shared_prefix_is_bounded_by_what_its_kernels_count(lib, seqs, q, width, group, apart):
    """Where its units would pass 32 bits a call goes sequence by sequence, and asks for no memory for parts."""
    heads = 8

    def together(width):
        pages, chunk = sizes(seqs, seqs * q, width, heads)
        options = _native.AttendOptions(A, None, 1, 0, 0)
        return lib.secure_infer_attend_parts(ct.byref(pages), ct.byref(chunk), group * heads, ct.byref(options)) > 0

    def units(width, row_cost, pair_cost):
        rows = seqs * q * group
        few = (seqs + 1) * 3 * heads * (width + row_cost)
        many = (2 * rows // (2 * (128 // group * group)) + seqs + 1) * heads * (width + pair_cost)
        return few if apart == "rows" else many

    assert units(width, 1, 2) < 2 ** 31 <= units(width, 2, 4)
    assert not together(width) and not together(width + 1)
    assert units(width - 3, 2, 4) < 2 ** 31 and together(width - 3)


CSRC = Path(__file__).resolve().parents[1] / "secure_infer_b200" / "csrc"


@pytest.mark.parametrize("function,arrays", [("find_seq", "cu"), ("load_any", "p.cu|p.kv|p.prefix|p.shared")])
def test_what_is_read_before_a_kernel_has_waited_comes_from_l2(function, arrays):
    """Lines that an earlier kernel on the SM left in L1 may be older than what the call was given."""
    text = re.sub(r"//[^\n]*", "", (CSRC / "paged.cuh").read_text())
    at = re.search(r"%s\([^;]*?\)\n\{" % function, text).end()
    body = text[at:text.index("\n}\n", at)]
    names = "|".join(re.escape(n) for n in arrays.split("|"))
    reads = re.findall(r"(?:__ldcg\((?:reinterpret_cast<const int4\*>\()?)?(?<![\w.])(?:%s)(?![\w.])" % names, body)
    assert reads and all(r.startswith("__ldcg(") for r in reads), reads
