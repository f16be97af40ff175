"""Operators on the paged KV cache that reloads fill (include/secure_infer_paged.h).

* ``append``  -- rotary positions (one or several axes) of a step's new queries
  and keys, and the new keys' and values' way into their pages;
* ``attend``  -- attention of the new tokens over the pages, from single tokens
  to long chunks, ragged over sequences;
* ``CachePages`` -- copies, forks, reserves, frees and compacts pages of all
  layers.

A layer's cache is K and V of ``[pages, 128, KV heads, 128]`` in bf16 or fp16,
as ``NativeTransfer`` and ``LayerwiseReloader`` fill it.  Handles
(``LayerPages``, ``CachePages``, ``Rotary``) are made once, a ``Chunk`` once per
step for all its layers.  Calls run on the current stream and return without
waiting; lengths, tables and page ids stay on the device (those given as lists are
copied there first, which does wait).  Bad arguments raise ``ValueError`` before
anything is launched, a refused launch ``RuntimeError``.  Outputs carry no gradient.
As everywhere in this package there is no fallback: the work goes through
``libsecure_infer.so``, reached by a small extension (csrc/paged_python.cpp) that
also looks the tensors over; ``copy`` alone goes by ctypes.
"""
from __future__ import annotations

import ctypes as ct
import math
from typing import NamedTuple

import torch

from . import _native

PAGE = 128
HEAD_DIM = 128
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _ints(t, what: str, device, dims: int) -> torch.Tensor:
    """An int32 tensor of the device, as given or made from a list."""
    if not isinstance(t, torch.Tensor):
        t = torch.tensor(list(t), dtype=torch.int32, device=device)
    if t.dtype is not torch.int32 or t.ndim != dims or t.device != device:
        raise ValueError(f"{what} must be an int32 tensor of {dims} dimension(s) on {device}")
    if t.stride(-1) != 1 and t.numel() != 0:
        raise ValueError(f"{what} must be dense in its last dimension")
    return t


# Reading the current stream's handle costs a twentieth of building a Stream object, where torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(index: int, function, *args):
    """function(*args) with device `index` current."""
    if index == torch.cuda.current_device():
        return function(*args)
    with torch.cuda.device(index):
        return function(*args)


class LayerPages:
    """One layer's paged cache: ``k`` and ``v`` ``[pages, 128, heads, 128]`` of
    one type, in any order of pages, tokens and heads in memory."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        shape, dtype, device = k.shape, k.dtype, k.device
        if v.shape != shape or v.dtype is not dtype or v.device != device:
            raise ValueError("K and V differ in shape, type or device")
        if len(shape) != 4 or shape[0] == 0 or shape[1] != PAGE or shape[2] == 0 or shape[3] != HEAD_DIM:
            raise ValueError(f"a cache is [pages, {PAGE}, heads, {HEAD_DIM}], not {list(shape)}")
        if dtype not in _DTYPES:
            raise ValueError(f"a cache holds bf16 or fp16, not {dtype}")
        if not k.is_cuda:
            raise ValueError("the cache must be on a CUDA device")
        strides = []
        for t in (k, v):
            sp, st, sh, sd = t.stride()
            if shape[0] == 1:
                sp = PAGE * HEAD_DIM * shape[2]
            if shape[2] == 1:
                sh = HEAD_DIM
            if sd != 1 or t.data_ptr() & 15 or sp <= 0 or st <= 0 or sh <= 0 or (sp | st | sh) & 7:
                raise ValueError("a head's values must be adjacent, the cache's address and strides multiples of 16 bytes")
            strides.append((sp, st, sh))
        self.k, self.v = k, v
        self.pages, self.heads, self.dtype, self.device, self.index = shape[0], shape[2], dtype, device, device.index
        self._strides = tuple(strides)
        self._c = _native.Pages(k.data_ptr(), v.data_ptr(), strides[0], strides[1], self.pages, self.heads, _DTYPES[dtype], 0)
        self._address = ct.addressof(self._c)


class Chunk:
    """The new tokens of one step, ragged over its sequences.

    ``block_table`` int32 ``[seqs, width]``: page of every 128 tokens (entries
    past a sequence's length are not read); ``cu_q`` int32 ``[seqs + 1]``: where
    each sequence's new tokens begin; ``kv_lens`` int32 ``[seqs]``: its tokens in
    all, the new ones last.  ``max_q``: no sequence has more new tokens; given,
    it lets steps of single tokens take their own path.  The tensors are kept
    and read when the operators run, so a captured graph follows their contents.
    """

    def __init__(self, block_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, max_q: int | None = None):
        _need(isinstance(block_table, torch.Tensor) and block_table.is_cuda, "block_table must be on a CUDA device")
        device = block_table.device
        _ints(block_table, "block_table", device, 2)
        _ints(cu_q, "cu_q", device, 1)
        _ints(kv_lens, "kv_lens", device, 1)
        seqs, width = block_table.shape
        _need(seqs > 0 and width > 0, "block_table is empty")
        _need(cu_q.shape[0] == seqs + 1 and kv_lens.shape[0] == seqs, "cu_q needs seqs + 1 entries, kv_lens seqs")
        _need(max_q is None or max_q >= 0, "max_q is negative")
        stride = block_table.stride(0) if seqs > 1 else width
        _need(stride >= width, "block_table's rows overlap")
        self.block_table, self.cu_q, self.kv_lens, self.device = block_table, cu_q, kv_lens, device
        self._c = _native.Chunk(block_table.data_ptr(), cu_q.data_ptr(), kv_lens.data_ptr(), stride, width, seqs, 0,
                                max_q or 0)
        self._address = ct.addressof(self._c)


class Rotary:
    """Rotary positions of 128-value heads: pair ``i`` turns by ``position *
    base ** (-i / 64)`` radians.  ``sections``: how many of the 64 pairs, in
    order, go by each axis of the positions (``(64,)``: one axis; ``(16, 24,
    24)``: time, height, width).  ``interleaved``: pair ``i`` is elements ``2i``
    and ``2i + 1`` instead of ``i`` and ``i + 64``."""

    def __init__(self, base: float = 10000.0, sections=(64,), interleaved: bool = False, device="cuda"):
        sections = [int(n) for n in sections]
        _need(base > 0 and math.isfinite(base), "base must be positive")
        _need(len(sections) > 0 and all(n >= 0 for n in sections) and sum(sections) == HEAD_DIM // 2,
              f"sections must be counts that add up to {HEAD_DIM // 2}")
        self.axes, self.interleaved = len(sections), bool(interleaved)
        # Revolutions per position as a fraction of 2^64, so a position's angle is an exact product modulo one turn; the
        # axis of each pair behind them.
        turns = [round(base ** (-i / 64) / (2 * math.pi) * 2.0 ** 64) % (1 << 64) for i in range(HEAD_DIM // 2)]
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
        table = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns] +
                             [axis[i] | axis[i + 1] << 32 for i in range(0, HEAD_DIM // 2, 2)], dtype=torch.int64, device=device)
        self.phase, self.axis = table[:HEAD_DIM // 2], table[HEAD_DIM // 2:].view(torch.int32)
        self.device = table.device
        self._c = (self.phase.data_ptr(), self.axis.data_ptr(), self.axes, self.interleaved)


def _call(name: str, device, *args) -> None:
    if _on(device.index, getattr(_native.lib(), name), *args) != 0:
        raise RuntimeError(f"{name} refused its arguments or failed to launch")


def append(pages: LayerPages, chunk: Chunk, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, *,
           rotary: Rotary | None = None, positions: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """Write the chunk's ``k`` and ``v`` ``[tokens, heads, 128]`` into their
    pages, keys turned by ``rotary``; returns ``q`` ``[tokens, q heads, 128]``
    turned likewise (``out``, or a new tensor; ``None`` without ``q``).

    ``positions`` int32 ``[axes, tokens]`` or ``[tokens]``; by default the
    tokens' places in their sequences.  A token whose place lies outside its
    sequence's pages is not written."""
    if chunk.device != pages.device or (rotary is not None and rotary.device != pages.device):
        raise ValueError("the chunk, rotary and the cache are on different devices")
    phase, axis, axes, interleaved = (0, 0, 1, False) if rotary is None else rotary._c
    index = pages.index
    return _on(index, _native.paged_ops().append, pages._address, chunk._address, index, q, k, v, phase, axis, axes,
               interleaved, positions, out, _raw_stream(index))


_workspaces: dict = {}   # (device, stream): what the stream's own calls use
_captured: dict = {}     # (device, stream): the stream's latest capture and what its calls use
_STATE = 4096            # SECURE_INFER_ATTEND_STATE_BYTES


def _workspace_bytes(index: int) -> int:
    return int(_on(index, _native.lib().secure_infer_paged_attend_workspace))


def attend_workspace(device) -> torch.Tensor:
    """A workspace for ``attend`` (41 MB on a B200).  Calls that may run at the
    same time, on two streams or in a graph beside either, need one each."""
    device = torch.device(device)
    index = torch.cuda.current_device() if device.index is None else device.index
    return torch.zeros(_workspace_bytes(index), dtype=torch.uint8, device=torch.device("cuda", index))


def release_workspaces(stream: torch.cuda.Stream | None = None) -> None:
    """Give up the workspaces that ``attend`` keeps, of all streams or of one:
    before a stream is destroyed, since its handle may come back as another's.
    The next call makes a new one."""
    for kept in (_workspaces, _captured):
        for key in [k for k in kept if stream is None or k == (stream.device.index, stream.cuda_stream)]:
            del kept[key]


def _workspace(index: int, stream: int) -> torch.Tensor:
    capture = _native.paged_ops().capture_id(stream)
    if capture:
        # The graph's calls keep theirs wherever it is replayed, so it is the graph's own: from its memory, held until the
        # stream's next capture lest this one gives it to other tensors, cleared at every replay's first call.
        held, w = _captured.get((index, stream), (0, None))
        if held != capture:
            w = torch.empty(_workspace_bytes(index), dtype=torch.uint8, device=torch.device("cuda", index))
            w[:_STATE].zero_()
            _captured[index, stream] = capture, w
        return w
    w = _workspaces.get((index, stream))
    if w is None:
        w = _workspaces[index, stream] = attend_workspace(torch.device("cuda", index))
    return w


def attend(pages: LayerPages, chunk: Chunk, q: torch.Tensor, *, scale: float | None = None, causal: bool = True,
           window: int = 0, return_lse: bool = False, out: torch.Tensor | None = None,
           workspace: torch.Tensor | None = None):
    """Attention of the chunk's queries ``[tokens, q heads, 128]`` over the
    pages: query head ``h`` reads KV head ``h // (q heads / KV heads)``.

    ``scale``: of the scores, 128 ** -0.5 by default.  ``causal``: the token at
    position ``p`` sees keys ``0 .. p``, with ``window`` only the last
    ``window`` of them; otherwise all of its sequence.  Returns ``[tokens,
    q heads, 128]``, and with ``return_lse`` the natural logarithms of the
    softmax sums, float32 ``[tokens, q heads]``, to join it with attention over
    other keys.  A row that sees no key gives 0 and -inf; rows of tokens past
    the chunk's last are left as they were.  ``workspace``:
    ``attend_workspace(device)``, by default one that the current stream keeps
    for its calls, and while it is captured one of the graph's own."""
    if chunk.device != pages.device:
        raise ValueError("the chunk and the cache are on different devices")
    index = pages.index
    stream = _raw_stream(index)
    return _on(index, _native.paged_ops().attend, pages._address, chunk._address, index, q, out, return_lse,
               HEAD_DIM ** -0.5 if scale is None else scale, causal, window,
               _workspace(index, stream) if workspace is None else workspace, stream)


def attend_status(workspace: torch.Tensor | None = None) -> int:
    """0, or 1 if a wait inside ``attend`` ran out in a call with ``workspace``
    (by default the one that the current stream keeps).  Such a call leaves NaN
    in its rows, and so does every later one with this workspace until this has
    reported it.  Waits for the current stream."""
    _need(workspace is None or workspace.is_cuda, "workspace must come from attend_workspace")
    index = torch.cuda.current_device() if workspace is None else workspace.device.index
    stream = _raw_stream(index)
    if workspace is None:
        workspace = _workspaces.get((index, stream))
        if workspace is None:
            return 0
    status = ct.c_uint32()
    _call("secure_infer_attend_status", workspace.device, workspace.data_ptr(), ct.addressof(status), stream)
    return status.value


class _Tables(NamedTuple):
    block_table: torch.Tensor
    lens: torch.Tensor
    refs: torch.Tensor


class PageTables(_Tables):
    """Who holds which page: ``block_table`` int32 ``[seqs, width]``, ``lens``
    int32 ``[seqs]`` tokens held, ``refs`` int32 ``[pages]`` rows that hold a
    page (0: free).  A sequence of n tokens holds ``ceil(n / 128)`` pages."""


class CachePages:
    """The pages of a whole cache, ``kv_caches[layer] = [K, V]`` as
    ``LayerwiseReloader`` takes it; ``layers[l]`` is layer l's ``LayerPages``.

    The table operations return new tables and leave the given ones as they
    are, so work in flight may go on reading those."""

    def __init__(self, kv_caches):
        self.layers = [LayerPages(k, v) for k, v in kv_caches]
        _need(len(self.layers) > 0, "a cache has at least one layer")
        first = self.layers[0]
        self.pages, self.device = first.pages, first.device
        shape, size = first.k.shape, first.k.element_size()
        self.page_bytes = PAGE * first.heads * HEAD_DIM * size
        self._tensors = (_native.PageTensor * (2 * len(self.layers)))()
        dense = {}   # page strides of the layouts met so far
        for i, layer in enumerate(self.layers):
            if layer.k.shape != shape or layer.dtype is not first.dtype or layer.device != first.device:
                raise ValueError("the layers' caches differ in shape, type or device")
            for j, (t, strides) in enumerate(zip((layer.k, layer.v), layer._strides)):
                if strides not in dense:
                    page, token, head = strides
                    inner = (token, head) if first.heads == 1 else sorted((token, head))
                    fills = token == HEAD_DIM if first.heads == 1 else \
                        inner[0] == HEAD_DIM and inner[1] == HEAD_DIM * (first.heads if inner[0] == head else PAGE)
                    _need(fills and page * size >= self.page_bytes, "a page's values must fill one block of memory")
                    dense[strides] = page * size
                self._tensors[2 * i + j] = (t.data_ptr(), dense[strides])
        self._address = ct.addressof(self._tensors)

    def _run(self, name: str, tables: PageTables, out: PageTables | None, *args):
        """The new tables and what else an operation on tables returns."""
        _need(isinstance(tables, PageTables), "tables must be PageTables")
        index = self.device.index
        made = _on(index, getattr(_native.paged_ops(), name), *tables, self.pages, index, *args, _raw_stream(index), out)
        return (PageTables(*made[:3]) if out is None else out, *made[3:])

    def _pair(self, a, b, names) -> tuple[torch.Tensor, torch.Tensor]:
        a, b = _ints(a, names[0], self.device, 1), _ints(b, names[1], self.device, 1)
        if a.shape != b.shape:
            raise ValueError(f"{names[0]} and {names[1]} differ in length")
        return a, b

    def copy(self, src, dst) -> None:
        """Copy pages ``src[i]`` to ``dst[i]`` in every layer.  No page may be
        written twice, or written and read; pairs outside the cache are skipped.
        Lists are checked here, device tensors are the caller's to keep so."""
        if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            src, dst = [int(i) for i in src], [int(i) for i in dst]
            _need(len(set(dst)) == len(dst) and not set(dst) & set(src), "a page is written twice, or written and read")
            _need(all(0 <= i < self.pages for i in src + dst), "page outside the cache")
        src, dst = self._pair(src, dst, ("src", "dst"))
        _call("secure_infer_paged_copy", self.device, self._tensors, len(self._tensors), self.page_bytes, self.pages,
              src.data_ptr(), dst.data_ptr(), src.shape[0], _raw_stream(self.device.index))

    def fork(self, tables: PageTables, parents, children, out: PageTables | None = None):
        """Give the empty sequence ``children[i]`` the tokens of ``parents[i]``:
        it shares the full pages, and a partial last one is copied to the lowest
        free page in every layer.  Returns the new tables and ``granted`` int32
        ``[n]``: 0 where the child is not empty or named twice, an index is out
        of range, or pages ran out (requests are served in order)."""
        a, b = self._pair(parents, children, ("parents", "children"))
        return self._run("fork", tables, out, self._address, len(self._tensors), self.page_bytes, a, b)

    def reserve(self, tables: PageTables, seqs, lens, out: PageTables | None = None):
        """Grow sequence ``seqs[i]`` to ``lens[i]`` tokens on the lowest free
        pages.  Returns the new tables and ``granted`` int32 ``[n]``: 0 where it
        would shrink or not fit the table, is named twice, its partial last page
        is shared, or fewer pages are left than it needs (requests are served in
        order, and later ones may still have those)."""
        a, b = self._pair(seqs, lens, ("seqs", "lens"))
        return self._run("reserve", tables, out, a, b)

    def free(self, tables: PageTables, seqs, out: PageTables | None = None) -> PageTables:
        """Empty the sequences ``seqs``; a page that no other row holds becomes
        free.  Returns the new tables."""
        return self._run("free", tables, out, _ints(seqs, "seqs", self.device, 1))[0]

    def compact(self, tables: PageTables, out: PageTables | None = None):
        """Move the used pages to the lowest places, in every layer: with
        ``live`` pages in use, the i-th used page at or above ``live`` goes to
        the i-th free one below.  Returns the new tables, ``moved`` int32
        ``[pages]`` (where each page is now, -1 for a free one) and ``live``
        int32 ``[1]``."""
        return self._run("compact", tables, out, self._address, len(self._tensors), self.page_bytes)
