"""The paged-cache operators' C ABI and bindings where there is no GPU: every
declared function is bound, and bad arguments come back as errors."""
from __future__ import annotations

import ctypes as ct
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from secure_infer_b200 import _native, paged

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def test_every_declaration_is_exported_and_bound(lib):
    text = (ROOT / "include" / "secure_infer_paged.h").read_text()
    names = set(re.findall(r"^(?:int|uint64_t) (secure_infer_paged_\w+)\(", text, re.M))
    assert len(names) == 9 and names == set(_native.PAGED_SIGNATURES)
    assert all(hasattr(lib, n) for n in names)


def test_structures_match_the_header():
    text = (ROOT / "include" / "secure_infer_paged.h").read_text()
    for name, cls in (("pages", _native.Pages), ("chunk", _native.Chunk), ("tables", _native.Tables),
                      ("page_tensor", _native.PageTensor)):
        body = text[:text.index("} secure_infer_%s;" % name)].rsplit("typedef struct {", 1)[1]
        fields = re.findall(r"(\w+)(?:\[3\])?;", body)
        assert fields == [f for f, _ in cls._fields_], name


# Addresses that are never read: every call below is refused before a launch.
A = 1 << 20


def good():
    pages = _native.Pages(A, A, (ct.c_int64 * 3)(131072, 1024, 128), (ct.c_int64 * 3)(131072, 1024, 128), 10, 8, 0, 0)
    chunk = _native.Chunk(A, A, A, 4, 4, 2, 3, 1)
    return pages, chunk, (ct.c_int64 * 2)(4096, 128)


@pytest.mark.parametrize("change", [
    lambda p, c, s: setattr(p, "k", None), lambda p, c, s: setattr(p, "v", A + 8), lambda p, c, s: setattr(p, "pages", 0),
    lambda p, c, s: setattr(p, "heads", 0), lambda p, c, s: setattr(p, "heads", 3), lambda p, c, s: setattr(p, "dtype", 2),
    lambda p, c, s: p.k_stride.__setitem__(1, 1023), lambda p, c, s: p.v_stride.__setitem__(0, -131072),
    lambda p, c, s: setattr(c, "block_table", None), lambda p, c, s: setattr(c, "cu_q", None),
    lambda p, c, s: setattr(c, "kv_lens", None), lambda p, c, s: setattr(c, "seqs", 0),
    lambda p, c, s: setattr(c, "table_width", 5), lambda p, c, s: setattr(c, "tokens", 1 << 30),
    lambda p, c, s: s.__setitem__(0, 4097), lambda p, c, s: s.__setitem__(1, 0),
])
def test_attend_and_append_refuse(lib, change):
    pages, chunk, stride = good()
    change(pages, chunk, stride)
    assert lib.secure_infer_paged_attend(ct.byref(pages), ct.byref(chunk), A, *stride, 32, A, None, 1.0, 1, 0, A, None) == -1
    if pages.heads != 3:   # any head count of its own goes with append
        assert lib.secure_infer_paged_append(ct.byref(pages), ct.byref(chunk), A, *stride, 32, A, A, *stride, A, *stride,
                                             None, None, None, 0, 1, 0, None) == -1


def test_attend_refuses_more(lib):
    pages, chunk, stride = good()
    call = lib.secure_infer_paged_attend
    p, c = ct.byref(pages), ct.byref(chunk)
    assert call(None, c, A, *stride, 32, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, None, A, *stride, 32, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, None, *stride, 32, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, A, 4096, -128, 32, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, A, *stride, 0, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, A, *stride, 33, A, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, A, *stride, 32, A + 2, None, 1.0, 1, 0, A, None) == -1
    assert call(p, c, A, *stride, 32, A, None, 1.0, 0, 9, A, None) == -1      # a window needs the causal order
    assert call(p, c, A, *stride, 32, A, None, 1.0, 1, 0, None, None) == -1
    assert call(p, c, A, *stride, 32, A, None, 1.0, 1, 0, A + 16, None) == -1
    chunk.tokens = 0
    assert call(p, c, None, *stride, 32, None, None, 1.0, 1, 0, A, None) == 0   # nothing to do
    assert lib.secure_infer_paged_attend_workspace() > 0


def test_append_refuses_more(lib):
    pages, chunk, stride = good()
    p, c = ct.byref(pages), ct.byref(chunk)

    def call(q=A, k=A, v=A, out=A, qs=stride, heads=32, phase=None, axis=None, positions=None, pos_stride=0, axes=1):
        return lib.secure_infer_paged_append(p, c, q, *qs, heads, out, k, *stride, v, *stride, phase, axis, positions,
                                             pos_stride, axes, 0, None)
    assert call(k=None) == -1 and call(v=A + 2) == -1 and call(q=A + 4) == -1 and call(out=None) == -1
    assert call(qs=(4096, 0)) == -1 and call(heads=0) == -1
    assert call(phase=A) == -1 and call(axis=A) == -1
    assert call(phase=A, axis=A, positions=A, axes=0) == -1 and call(phase=A, axis=A, positions=A, pos_stride=-1) == -1
    chunk.tokens = 0
    assert call(k=None) == 0


def test_table_calls_refuse(lib):
    a, b = _native.Tables(A, A, A, 4, 4, 9, 0), _native.Tables(2 * A, 2 * A, 2 * A, 4, 4, 9, 0)
    t = (_native.PageTensor * 1)()
    t[0].base, t[0].page_stride = A, 32768
    tensors = (t, 1, 32768)
    assert lib.secure_infer_paged_scratch(ct.byref(a), 7) >= 4 * (2 * 9 + 2 * 4 + 7)
    assert lib.secure_infer_paged_scratch(None, 7) == 0
    for x, y in ((None, ct.byref(b)), (ct.byref(a), None), (ct.byref(a), ct.byref(a))):
        assert lib.secure_infer_paged_free(x, y, A, 1, A, None) == -1
        assert lib.secure_infer_paged_reserve(x, y, A, A, 1, A, A, None) == -1
        assert lib.secure_infer_paged_fork(*tensors, x, y, A, A, 1, A, A, None) == -1
        assert lib.secure_infer_paged_compact(*tensors, x, y, A, A, A, None) == -1
    other = _native.Tables(2 * A, 2 * A, 2 * A, 4, 5, 9, 0)
    assert lib.secure_infer_paged_free(ct.byref(a), ct.byref(other), A, 1, A, None) == -1
    ok = (ct.byref(a), ct.byref(b))
    assert lib.secure_infer_paged_free(*ok, None, 1, A, None) == -1
    assert lib.secure_infer_paged_free(*ok, A, 1, None, None) == -1
    assert lib.secure_infer_paged_fork(*tensors, *ok, None, A, 1, A, A, None) == -1
    assert lib.secure_infer_paged_compact(*tensors, *ok, None, A, A, None) == -1
    for bad in ((None, 1, 32768), (t, 0, 32768), (t, 1, 0), (t, 1, 24), (t, 1, 65536)):
        assert lib.secure_infer_paged_copy(*bad, 9, A, A, 1, None) == -1
    assert lib.secure_infer_paged_copy(*tensors, 9, None, A, 1, None) == -1
    assert lib.secure_infer_paged_copy(*tensors, 9, None, None, 0, None) == 0
    t[0].base = A + 8
    assert lib.secure_infer_paged_copy(*tensors, 9, A, A, 1, None) == -1


def test_python_refuses_host_tensors():
    k = torch.zeros((3, 128, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.LayerPages(k, k)
    with pytest.raises(ValueError, match="CUDA"):
        paged.Chunk(torch.zeros((1, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="pages"):
        paged.LayerPages(k[:, :64], k[:, :64])
    with pytest.raises(ValueError):
        paged.Rotary(sections=(1, 2), device="cpu")


def test_rotary_phases_are_exact_fractions_of_a_turn():
    """position * phase modulo 2^64 against the angle in 50 digits."""
    from decimal import Decimal, getcontext
    getcontext().prec = 50
    pi = Decimal("3.14159265358979323846264338327950288419716939937510")
    r = paged.Rotary(base=500000.0, sections=(16, 24, 24), device="cpu")
    assert r.axis.tolist() == [0] * 16 + [1] * 24 + [2] * 24
    for i in (0, 1, 17, 40, 63):
        phase = r.phase[i].item() % (1 << 64)
        for pos in (1, 127, 100003, (1 << 20) + 7):
            turns = Decimal(pos) * (Decimal(500000) ** (Decimal(-i) / 64)) / (2 * pi)
            want = turns - int(turns)
            got = Decimal((pos * phase) % (1 << 64)) / Decimal(1 << 64)
            off = abs(got - want)
            assert min(off, 1 - off) < Decimal("1e-9")   # 2^-53 of the phase times 2^20 positions


def test_extension_refuses_before_any_launch():
    """The calls of every layer look their arguments over in the extension."""
    ops = _native.paged_ops()
    with pytest.raises(TypeError):
        ops.attend(1, 2)
    pages, chunk, _ = good()
    p, c = ct.addressof(pages), ct.addressof(chunk)
    q = torch.zeros((3, 32, 128), dtype=torch.bfloat16)
    for bad in (q, q[:, :, :64], q.float(), q[0], None, 7):
        with pytest.raises(ValueError):
            ops.attend(p, c, 0, bad, None, False, 1.0, True, 0, None, 0)
        with pytest.raises(ValueError):
            ops.append(p, c, 0, None, bad, bad, 0, 0, 1, False, None, None, 0)
    t = torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.free(t, t[0], t[0], 2, 0, t[0], 0)


def test_extension_missing_is_said(monkeypatch, tmp_path):
    monkeypatch.setattr(_native, "_paged", None)
    monkeypatch.setattr(_native, "LIB_PATH", tmp_path / "libsecure_infer.so")
    with pytest.raises(_native.NativeLibraryMissing, match="paged_python"):
        _native.paged_ops()


def test_status_refuses(lib):
    word = ct.c_uint32(7)
    call = lib.secure_infer_attend_status
    assert call(None, ct.byref(word), None) == -1
    assert call(A + 16, ct.byref(word), None) == -1
    assert call(A, None, None) == -1
    assert word.value == 7


def test_attend_fits_by_what_is_launched(lib):
    """Units of work are a page for a tile: of 256 rows where there are more than a few, of eight otherwise."""
    pages, chunk, _ = good()

    def fits(tokens, max_q, width, seqs=1, heads=32, kv_heads=8):
        pages.heads, chunk.tokens, chunk.max_q, chunk.seqs = kv_heads, tokens, max_q, seqs
        chunk.table_width = chunk.table_stride = width
        return lib.secure_infer_attend_fits(ct.byref(pages), ct.byref(chunk), heads)

    assert fits(2, 1, 4, 2)
    assert fits(65536, 0, 8192, heads=64)                  # a long prompt in a table for a million tokens
    assert fits(65536, 0, 8192, 64, heads=64)
    assert fits(2048, 0, 1 << 20) and fits(2048, 0, 1 << 22)
    assert not fits(2048, 0, 1 << 22, heads=64, kv_heads=64)
    assert not fits(1 << 20, 1, 1 << 12, 1 << 20)          # a million single tokens
    assert fits(1 << 12, 1, 1 << 12, 1 << 12)
    assert not fits(1 << 28, 0, 4, heads=4096)             # rows beyond 32 bits
    assert not fits(4, 1, 1 << 24)                         # wider than a table may be
    assert not fits(4, 1, 4, heads=33)
    assert not lib.secure_infer_attend_fits(None, ct.byref(chunk), 32)
    assert not lib.secure_infer_attend_fits(ct.byref(pages), None, 32)
