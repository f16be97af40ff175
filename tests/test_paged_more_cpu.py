"""Refusals of attention with sinks and shared prefixes, of joining and of
trimming, where there is no GPU: bad arguments come back before any launch."""
from __future__ import annotations

import ctypes as ct
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from secure_infer_b200 import _native, paged

ROOT = Path(__file__).resolve().parents[1]
A = 1 << 20   # an address that is never read


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def good():
    pages = _native.Pages(A, A, (ct.c_int64 * 3)(131072, 1024, 128), (ct.c_int64 * 3)(131072, 1024, 128), 10, 8, 0, 0)
    return pages, _native.Chunk(A, A, A, 4, 4, 2, 3, 1)


def test_every_declaration_is_exported_and_bound(lib):
    text = (ROOT / "include" / "secure_infer_paged.h").read_text()
    names = set(re.findall(r"^(?:int|uint64_t) (secure_infer_\w+)\(", text, re.M))
    assert {"secure_infer_attend", "secure_infer_attend_parts", "secure_infer_attend_join",
            "secure_infer_shared_prefix", "secure_infer_shared_prefix_ints", "secure_infer_trim"} <= names
    assert names <= set(_native.HOST_SIGNATURES) and all(hasattr(lib, n) for n in names)


def test_structures_match_the_header():
    text = (ROOT / "include" / "secure_infer_paged.h").read_text()
    for name, cls in (("attend_options", _native.AttendOptions), ("attend_part", _native.AttendPart)):
        body = text[:text.index("} secure_infer_%s;" % name)].rsplit("typedef struct {", 1)[1]
        assert re.findall(r"(\w+)(?:\[2\])?;", body) == [f for f, _ in cls._fields_], name


@pytest.mark.parametrize("window,causal,options", [
    (0, 1, (None, None, 0, 0, 4)),        # sinks without a window
    (8, 0, (None, None, 0, 0, 4)),        # a window without the causal order
    (8, 1, (None, None, 0, 0, 1 << 31)),
    (8, 1, (A, A, 1, 0, 0)),              # a shared prefix with a window
    (0, 1, (A, A, 0, 0, 0)),              # no group
    (0, 1, (A, A, 65, 0, 0)),             # more groups than sequences
    (0, 1, (A + 4, A, 1, 0, 0)),
    (0, 1, (A, None, 1, 0, 0)),
    (0, 1, (A, A + 8, 1, 0, 0)),
])
def test_attend_refuses(lib, window, causal, options):
    pages, chunk = good()
    chunk.seqs, chunk.tokens, chunk.table_width, chunk.table_stride = 64, 64, 1000, 1000
    o = _native.AttendOptions(*options)
    assert lib.secure_infer_attend(ct.byref(pages), ct.byref(chunk), A, 4096, 128, 32, A, None, 1.0, causal, window, ct.byref(o),
                                   A, None) == -1
    chunk.tokens = 0
    if options[1] is None and options[0] is not None:   # parts are only needed where there are tokens
        assert lib.secure_infer_attend(ct.byref(pages), ct.byref(chunk), None, 4096, 128, 32, None, None, 1.0, 1, 0, ct.byref(o),
                                       A, None) == 0


def test_what_is_shared_by_its_sizes(lib):
    """Memory for parts is asked for where the groups' pages are attended together: by what that saves."""
    pages, chunk = good()

    def parts(seqs, q, width, groups=1, heads=32, kv_heads=8, common=0, max_q=None):
        pages.heads, chunk.tokens, chunk.max_q, chunk.seqs = kv_heads, seqs * q, q if max_q is None else max_q, seqs
        chunk.table_width = chunk.table_stride = width
        o = _native.AttendOptions(A, None, groups, common, 0)
        got = lib.secure_infer_attend_parts(ct.byref(pages), ct.byref(chunk), heads, ct.byref(o))
        assert got in (0, seqs * q * heads * 2 * 130 * 4)
        return got > 0

    assert parts(48, 1, 72) and not parts(2, 1, 6) and not parts(8, 1, 6)
    assert parts(24, 5, 240, 4, 8, 1) and not parts(24, 5, 240, 24, 8, 1)      # groups of one save nothing
    assert not parts(5, 300, 52, heads=28, kv_heads=4)                          # chunks that fill tiles of their own
    assert parts(48, 1, 4096) and not parts(48, 1, 4096, common=128) and parts(48, 1, 4096, common=1 << 20)
    assert not parts(1 << 17, 1, 1 << 12) and parts(1 << 14, 1, 1 << 10)        # units beyond 32 bits: sequence by sequence
    assert not parts(1, 1, 4096) and not parts(4, 0, 4096)
    o = _native.AttendOptions(None, None, 0, 0, 4)
    assert lib.secure_infer_attend_parts(ct.byref(pages), ct.byref(chunk), 32, ct.byref(o)) == 0
    assert lib.secure_infer_attend_parts(ct.byref(pages), ct.byref(chunk), 32, None) == 0
    assert lib.secure_infer_attend_parts(None, ct.byref(chunk), 32, ct.byref(o)) == 0
    assert lib.secure_infer_shared_prefix_ints(5, 2) == 8 + 8


def test_shared_prefix_refuses(lib):
    _, chunk = good()
    call = lib.secure_infer_shared_prefix
    assert call(None, A, 1, A, None) == -1
    assert call(ct.byref(chunk), A, 0, A, None) == -1
    assert call(ct.byref(chunk), A, 3, A, None) == -1
    assert call(ct.byref(chunk), None, 2, A, None) == -1
    assert call(ct.byref(chunk), A, 1, None, None) == -1
    assert call(ct.byref(chunk), A, 1, A + 8, None) == -1
    chunk.kv_lens = None
    assert call(ct.byref(chunk), A, 1, A, None) == -1


def test_join_refuses(lib):
    def call(n=2, tokens=3, heads=4, dtype=0, out=A, lse=A, part=(A, A, (512, 128), (4, 1)), parts=True):
        p = (_native.AttendPart * 8)()
        for i in range(8):
            p[i].out, p[i].lse = part[0], part[1]
            p[i].out_stride[:], p[i].lse_stride[:] = part[2], part[3]
        return lib.secure_infer_attend_join(p if parts else None, n, tokens, heads, dtype, out, lse, None)

    for bad in (dict(n=0), dict(n=9), dict(heads=0), dict(heads=1 << 17), dict(tokens=1 << 29), dict(dtype=2), dict(out=None),
                dict(out=A + 2), dict(lse=None), dict(parts=False), dict(part=(None, A, (512, 128), (4, 1))),
                dict(part=(A, None, (512, 128), (4, 1))), dict(part=(A, A, (511, 128), (4, 1))),
                dict(part=(A, A, (512, 0), (4, 1))), dict(part=(A, A, (512, 128), (-4, 1))),
                dict(part=(A, A, (512, 128), (4, -1))), dict(tokens=1 << 28, heads=1 << 16)):
        assert call(**bad) == -1, bad
    assert call(tokens=0, out=None) == 0


def test_trim_refuses(lib):
    a, b = _native.Tables(A, A, A, 4, 4, 9, 0), _native.Tables(2 * A, 2 * A, 2 * A, 4, 4, 9, 0)
    call = lib.secure_infer_trim
    ok = (ct.byref(a), ct.byref(b))
    assert call(None, ok[1], A, 1, 8, 0, A, None) == -1
    assert call(ok[0], ok[0], A, 1, 8, 0, A, None) == -1
    assert call(*ok, None, 1, 8, 0, A, None) == -1
    assert call(*ok, A, 1, 8, 0, None, None) == -1
    assert call(*ok, A, 1, 0, 0, A, None) == -1
    assert call(*ok, A, 1, 1 << 31, 0, A, None) == -1
    assert call(*ok, A, 1, 8, (1 << 31) - 2, A, None) == -1


def test_extension_and_python_refuse():
    ops = _native.paged_ops()
    pages, chunk = good()
    p, c = ct.addressof(pages), ct.addressof(chunk)
    q = torch.zeros((3, 32, 128), dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.attend(p, c, 0, q, None, False, 1.0, True, 0, None, 0, 4)
    with pytest.raises(ValueError):
        ops.attend(p, c, 0, q, None, False, 1.0, True, 0, None, 0, 4, None, 0, 0)
    lse = torch.zeros((3, 32))
    for bad in (((q, q), (lse,)), ((), ()), ((q,) * 9, (lse,) * 9), ((q, q), (lse, lse)), ((q, 3), (lse, lse)), ([q], [lse])):
        with pytest.raises(ValueError):
            ops.join(*bad, 0, None, 0)
    with pytest.raises(ValueError, match="CUDA"):
        paged.join([q, q], [lse, lse])
    with pytest.raises(ValueError):
        paged.join([], [])
    with pytest.raises(ValueError, match="Chunk"):
        paged.SharedPrefix(None)
    t = torch.zeros((2, 2), dtype=torch.int32)
    for window, sinks in ((0, 0), (-1, 0), (1 << 31, 0), (5, -1), (5, 1 << 31), (5, 0)):
        with pytest.raises(ValueError):
            ops.trim(t, t[0], t[0], 2, 0, t[0], window, sinks, 0, None)
