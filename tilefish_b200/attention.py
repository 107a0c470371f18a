"""The attention half of a decoder layer: rotary positions, a paged key-value cache, and attention of new tokens over it.

Three operators in the manner of ``kernels.py`` (torch tensors in, C ABI calls out, every precondition checked before anything is enqueued):

* ``rotary``           turns [tokens, heads, head_dim] by their positions (or back: ``inverse``, which is also its gradient);
* ``cache_append``     writes keys and values of new tokens into a ``PagedCache`` (bf16 or e4m3 entries), turning k and q on the way;
* ``paged_attention``  attention of the last tokens of each sequence over the cache, split over its length.

``attention_block`` puts them between the qkv and the output GEMM (residual_add_rmsnorm -> gemm -> cache_append -> paged_attention -> gemm), and
``decoder_layer`` puts that in front of ``mlp.decoder_block``. The reference has no counterpart: its README's graphs stop at the MLP block
(README.md:53-85).
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from fractions import Fraction
from typing import Optional

from . import _native as N
from . import kernels as K
from .kernels import _check, _dense, _pre, _stream, _torch

LAYOUTS = {"half": N.ROTARY_HALF, "interleaved": N.ROTARY_INTERLEAVED}
_TURN = round(2**192 / (2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")))  # 2^64 / 2 pi, times 2^128


# A call's checks run in front of launches of a few microseconds: shape, strides and address of a tensor are asked for once and device indexes are
# compared, and only a check that fails looks for what to say (a rotation of four tokens 14 -> 12 us a call).


def _strides(shape, strides):
    """The first two axes' strides, 0 for one that is never stepped along (its stride says nothing then)."""
    return strides[0] if shape[0] > 1 else 0, strides[1] if shape[1] > 1 else 0


def _here(index: int) -> None:
    current = _torch()._C._cuda_getDevice()
    if index != current:
        _pre(False, f"the tensors are on cuda:{index}, the current device is cuda:{current}: make it current (with torch.cuda.device(...))", "device")


def _rows(t, name: str, dtype, index: Optional[int], unit: int, align: int):
    """(shape, token stride, head stride, address) of a [tokens, heads, dim] tensor of ``dtype`` on device ``index`` (None: any): the last axis dense, the
    others at strides that are multiples of ``unit`` elements."""
    if not (isinstance(t, _torch().Tensor) and t.is_cuda and t.dtype == dtype and t.dim() == 3 and (index is None or t.get_device() == index)):
        _check(t, name, dtype, 3, None if index is None else _torch().device("cuda", index), align)
    shape, strides, at = t.shape, t.stride(), t.data_ptr()
    st, sh = _strides(shape, strides)
    if (strides[2] != 1 and shape[2] > 1) or st % unit or sh % unit or at % align:
        _pre(shape[2] <= 1 or strides[2] == 1, f"{name}: the last axis must be dense (strides {tuple(strides)})", "contiguous", name)
        _pre(st % unit == 0 and sh % unit == 0, f"{name}: strides {tuple(strides)} must be multiples of {unit} elements", "alignment", name)
        _pre(t.numel() == 0 or at % align == 0, f"{name}: the data pointer is not {align}-byte aligned", "pointer_alignment", name)
    return shape, st, sh, at


def _ints(t, name: str, n: Optional[int], index: int) -> int:
    """The address of a dense int32 [n] tensor."""
    torch = _torch()
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1 and t.get_device() == index and t.shape[0] == n and (n <= 1 or t.stride(0) == 1)):
        _check(t, name, torch.int32, 1, torch.device("cuda", index), align=4)
        _pre(t.shape[0] == n, f"{name}: {t.shape[0]} of them, expected {n}", "shape", name)
        _dense(t, name)
    return t.data_ptr()


def _span(t):
    """(first, behind the last) address of a tensor that has elements."""
    at = t.data_ptr()
    return at, at + (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size()


def _meet(apart: int, axes) -> bool:
    """Whether two boxes of ``axes`` (stride, lengths in the one and in the other; falling strides, none shorter than what the axes behind it reach) share an
    element when they begin ``apart`` of each other."""
    if not axes:
        return apart == 0
    stride, na, nb = axes[0]
    steps = apart // stride  # what is left over lies between two steps
    return any(-nb < d < na and _meet(apart - d * stride, axes[1:]) for d in (steps, steps + 1))


def _overlap(a, b) -> bool:
    """Whether two tensors of one rank and a dense last axis share memory. Slices of one tensor with all its strides do not; of tensors whose strides differ,
    or that overlap themselves, the whole ranges are compared."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    size, axes = a.element_size(), [(1, a.shape[-1] * a.element_size(), b.shape[-1] * b.element_size())]
    for na, nb, sa, sb in zip(a.shape[:-1], b.shape[:-1], a.stride(), b.stride()):
        na, nb = na if sa else 1, nb if sb else 1  # a broadcast axis is one element
        if na > 1 or nb > 1:
            if na > 1 and nb > 1 and sa != sb:
                return True
            axes.append(((sa if na > 1 else sb) * size, na, nb))
    axes.sort()
    reach = [0, 0]
    for stride, *n in axes:
        if stride < max(reach):
            return True
        reach = [r + stride * (m - 1) if r else m for r, m in zip(reach, n)]
    return _meet(b0 - a0, axes[::-1])


def _columns(a, b, size: int) -> bool:
    """Whether two [tokens, heads, dim] tensors, as ``_rows`` gives them, are columns of one matrix that do not meet: what slices of a qkv product are. Most calls with a
    result of the caller's need no other look (an append in place 13 us a call; with ``_overlap`` alone 31)."""
    (_, ha, dim), step, sa, a0 = a
    (_, hb, _), other, sb, b0 = b
    if step != other or step <= 0:
        return False
    wide_a, wide_b, apart = sa * (ha - 1) + dim, sb * (hb - 1) + dim, (b0 - a0) // size % step
    return wide_a <= apart and apart + wide_b <= step


def _ends(rows, size: int):
    """``_span`` of what ``_rows`` gives."""
    (tokens, heads, dim), st, sh, at = rows
    return at, at + ((tokens - 1) * st + (heads - 1) * sh + dim) * size


def _result(t, name: str) -> None:
    """No two elements of a [tokens, heads, dim] result are one: no stride 0, and one of the first two axes lies inside a step of the other."""
    (tokens, heads, dim), (st, sh, _) = t.shape, t.stride()
    if tokens and heads and not ((heads == 1 or sh >= dim) and (tokens == 1 or st >= (sh * (heads - 1) + dim)) or (tokens == 1 or st >= dim) and (heads == 1 or sh >= st * (tokens - 1) + dim)):
        _pre(False, f"{name}: elements share memory (strides {tuple(t.stride())}): a broadcast or overlapping view cannot be written", "alias", name)


def _apart(lo: int, hi: int, name: str, others) -> None:
    """The range of what a call writes shares nothing with those of ``others`` (span, name)."""
    for span, other in others:
        if lo < span[1] and span[0] < hi:
            _pre(False, f"{name} overlaps {other}", "alias", name)


# ---- rotary positions ---------------------------------------------------------------------------------------------------------


def _turns(frequencies):
    """Frequencies (radians per position) as the fraction of a full turn per position, times 2^64, in two's complement: exact integer arithmetic, rounded once."""
    out = []
    for f in frequencies:
        n, d = f.as_integer_ratio()  # d is a power of two
        turns = (2 * n * _TURN + (d << 128)) // (d << 129) & (2**64 - 1)
        out.append(turns - 2**64 if turns >= 2**63 else turns)
    return out


class RotaryTable:
    """What a rotation needs besides positions: one inverse frequency per pair, how pairs lie in a head, and what the result is multiplied by.

    ``inv_freq``   radians per position, rot / 2 of them (a tensor or a sequence; taken in 64 bits, read on the host once, here)
    ``layout``     "half": pairs (i, i + rot / 2); "interleaved": pairs (2i, 2i + 1)
    ``magnitude``  factor of the turned elements (long-context scalings use it); elements from rot on are left alone

    Made once per set of frequencies, and not while a CUDA graph is captured: frequencies on the device are waited for, and the table is copied there.
    """

    __slots__ = ("rot", "layout", "magnitude", "turns", "index", "_layout")

    def __init__(self, inv_freq, *, layout: str = "half", magnitude: float = 1.0, device=None) -> None:
        torch = _torch()
        _pre(layout in LAYOUTS, f"unknown layout {layout!r}: one of {sorted(LAYOUTS)}", "argument", "layout")
        _pre(abs(magnitude) <= 2.0**127, f"magnitude: {magnitude} is not a finite float32", "argument", "magnitude")
        if isinstance(inv_freq, torch.Tensor):
            _pre(inv_freq.dim() == 1, f"inv_freq: expected rank 1, got {inv_freq.dim()}", "rank", "inv_freq")
            if device is None and inv_freq.is_cuda:
                device = inv_freq.device
            inv_freq = inv_freq.double().tolist()
        values = [float(f) for f in inv_freq]
        _pre(1 <= len(values) <= 512, f"inv_freq: {len(values)} frequencies; 1 to 512 are possible", "shape", "inv_freq")
        _pre(all(abs(f) <= 2.0**32 for f in values), "inv_freq: not finite, or more than 2^32 radians", "argument", "inv_freq")
        turns = torch.tensor(_turns(values), dtype=torch.int64, device=device if device is not None else "cuda")
        for name, value in zip(RotaryTable.__slots__, (2 * len(values), layout, float(magnitude), turns, turns.get_device(), LAYOUTS[layout]), strict=True):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value) -> None:
        if name in RotaryTable.__slots__:
            raise AttributeError(f"RotaryTable.{name} cannot be exchanged: other frequencies, layouts or magnitudes are another table")
        object.__setattr__(self, name, value)

    def __setstate__(self, state) -> None:
        for part in state:
            for name, value in (part or {}).items():
                object.__setattr__(self, name, value)

    def __repr__(self) -> str:
        return f"RotaryTable(rot={self.rot}, {self.layout}, magnitude={self.magnitude:g})"


def rotary_frequencies(rot: int, *, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0, length: int = 0, low: float = 1.0,
                       high: Optional[float] = None):
    """(inverse frequencies, magnitude) for heads of which ``rot`` elements are turned: base^(-2i / rot), stretched for contexts ``factor`` times
    as long as the ``length`` a model was trained on:

    * "linear"  every frequency divided by ``factor``;
    * "ntk"     the base raised so that the lowest frequency is divided by ``factor`` and the highest is kept;
    * "bands"   frequencies that make fewer than ``low`` turns over ``length`` divided by ``factor``, those above ``high`` (4) kept, blended between
                by their number of turns;
    * "yarn"    the same kept and divided ends (``high`` 32), blended by index (Peng et al., "YaRN", 2023), with magnitude 0.1 ln(factor) + 1.
    """
    _pre(rot >= 2 and rot % 2 == 0, f"rot={rot} must be even and at least 2", "divisible", "rot")
    _pre(base > 0 and factor >= 1, f"base={base} must be positive and factor={factor} at least 1", "argument", "factor")
    _pre(scaling in (None, "linear", "ntk", "bands", "yarn"), f"unknown scaling {scaling!r}", "argument", "scaling")
    half = rot // 2
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    inv = [base ** (-2.0 * i / rot) for i in range(half)]
    if scaling == "linear" or (scaling == "ntk" and rot == 2):
        return [f / factor for f in inv], 1.0
    if scaling in (None, "ntk"):
        return inv, 1.0
    high = (4.0 if scaling == "bands" else 32.0) if high is None else high
    _pre(length > 0 and 0 < low < high, f"scaling {scaling!r} needs length > 0 and 0 < low < high (length={length}, low={low}, high={high})", "argument", "length")
    _pre(scaling == "bands" or base > 1, f"base={base}: scaling 'yarn' needs frequencies that fall from pair to pair, so more than 1", "argument", "base")
    if scaling == "bands":
        keep = [min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low))) for f in inv]
        return [f * (k + (1 - k) / factor) for f, k in zip(inv, keep)], 1.0

    def index_of(turns: float) -> float:  # the index whose frequency makes so many turns over `length`
        return rot * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

    # The line between the ends may go on behind the last pair (the method stops it at rot - 1): the slowest pair is then on it, or kept.
    last = min(rot - 1, math.ceil(index_of(low)))
    first = min(last - 1, max(0, math.floor(index_of(high))))
    keep = [1 - min(1.0, max(0.0, (i - first) / (last - first))) for i in range(half)]
    return [f * (k + (1 - k) / factor) for f, k in zip(inv, keep)], 0.1 * math.log(factor) + 1.0


def _check_positions(positions, tokens: int, index: int):
    """(address, 32 or 64)"""
    torch = _torch()
    if isinstance(positions, torch.Tensor) and positions.dtype == torch.int64:
        if not (positions.dim() == 1 and positions.get_device() == index and positions.shape[0] == tokens and (tokens <= 1 or positions.stride(0) == 1)):
            _check(positions, "positions", torch.int64, 1, torch.device("cuda", index), align=8)
            _pre(positions.shape[0] == tokens, f"positions: {positions.shape[0]} of them for {tokens} tokens", "shape", "positions")
            _dense(positions, "positions")
        return positions.data_ptr(), 64
    return _ints(positions, "positions", tokens, index), 32


def _check_table(table, dim: int, index: int) -> None:
    if not isinstance(table, RotaryTable):
        _pre(False, f"expected a RotaryTable, got {type(table).__name__}", "dtype", "table")
    if table.index != index:
        _pre(False, f"the table is on {table.turns.device}, the other arguments are on cuda:{index}", "device", "table")
    if table.rot > dim:
        _pre(False, f"the table turns {table.rot} elements of a head of {dim}", "shape", "table")


def rotary(x, positions, table: RotaryTable, *, out=None, inverse: bool = False, stream=None):
    """``x`` (bf16 or f32 [tokens, heads, head_dim], dense heads at any strides) with each token's heads turned by its position; f32 arithmetic, one rounding.
    ``inverse`` turns back by the same angle: the transposed map, so the gradient of ``rotary`` is ``rotary(grad, ..., inverse=True)``. ``out=x`` works in place.
    Positions are int32 or int64 of any size: an angle is exact to 2^-65 turns times the position, and rounded to f32 as its distance from the nearest
    quarter turn (2^-28 turns at the most)."""
    torch = _torch()
    f32 = isinstance(x, torch.Tensor) and x.dtype == torch.float32
    dtype, item = (torch.float32, 4) if f32 else (torch.bfloat16, 2)
    shape, st, sh, xp = _rows(x, "x", dtype, None, 1, item)
    tokens, heads, dim = shape
    index = x.get_device()
    _here(index)
    _check_table(table, dim, index)
    pp, bits = _check_positions(positions, tokens, index)
    if dim > 1024:
        _pre(False, f"x: head_dim {dim} is more than 1024", "unsupported", "x")
    if out is None:
        out = torch.empty_strided(shape, (heads * dim, dim, 1), dtype=dtype, device=x.device)
        ot, oh, op = heads * dim, dim, out.data_ptr()
    else:
        oshape, ot, oh, op = _rows(out, "out", dtype, index, 1, item)
        _pre(oshape == shape, f"out: shape {tuple(oshape)}, expected {tuple(shape)}", "shape", "out")
        _result(out, "out")
        _pre((op == xp and ot == st and oh == sh) or not _overlap(out, x), "out overlaps x without being x", "alias", "out")
    if tokens == 0 or heads == 0:
        return out
    N.check(N.load().tf_rotary(xp, N.TYPE_F32 if f32 else N.TYPE_BF16, tokens, heads, dim, st, sh, pp, bits, table.turns.data_ptr(), table.rot, table._layout,
                               table.magnitude, 1 if inverse else 0, op, ot, oh, _stream(stream)), "tf_rotary")
    return out


# ---- the paged cache ------------------------------------------------------------------------------------------------------------


class PagedCache:
    """Keys and values of many sequences in pages.

    ``k``, ``v``  [pages, kv_heads, page_size, head_dim], bf16, or uint8 holding e4m3 codes; the last axis dense, the others at any strides (the same for
                  both), so ``empty(...)``'s order and views of [pages, page_size, kv_heads, head_dim] tensors are both fine
    ``k_scale``, ``v_scale``  float32 [kv_heads] for e4m3 (an entry's value is code * scale; None: 1); not 0 and not below 2^-126

    Which pages belong to which sequence stands in the int32 [sequences, width] tables that the operators take, not here. The tensors' contents, scales included,
    may change between calls; other tensors are another cache (the operators go by the addresses that the cache was made with).
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "kv_heads", "page_size", "head_dim", "device", "index", "_desc", "_ref", "_spans")

    def __init__(self, k, v, k_scale=None, v_scale=None) -> None:
        torch = _torch()
        codes = isinstance(k, torch.Tensor) and k.dtype == torch.uint8
        dtype, unit = (torch.uint8, 16) if codes else (torch.bfloat16, 8)
        _check(k, "k", dtype, 4)
        _check(v, "v", dtype, 4, k.device)
        _pre(k.shape == v.shape, f"v: shape {tuple(v.shape)}, expected {tuple(k.shape)}", "shape", "v")
        _pre(min(k.shape) > 0, f"k: shape {tuple(k.shape)} has an empty axis", "shape", "k")
        pages, kv_heads, page_size, head_dim = k.shape
        _pre(head_dim % 16 == 0 and head_dim <= 256, f"k: head_dim {head_dim} is not a multiple of 16 up to 256", "divisible", "k")
        _pre(k.stride(3) == 1 and v.stride(3) == 1, "k, v: the last axis must be dense", "contiguous", "k")
        strides = [k.stride(i) if k.shape[i] > 1 else 0 for i in range(3)]
        _pre(strides == [v.stride(i) if v.shape[i] > 1 else 0 for i in range(3)], f"v: strides {tuple(v.stride())}, expected those of k, {tuple(k.stride())}", "contiguous", "v")
        _pre(all(s % unit == 0 for s in strides), f"k: strides {tuple(k.stride())} must be multiples of {unit} elements", "alignment", "k")
        axes = sorted((st, n) for st, n in zip(strides, k.shape[:3]) if n > 1)
        reach = head_dim
        for st, n in axes:
            _pre(st >= reach, f"k: strides {tuple(k.stride())}: entries overlap", "alias", "k")
            reach = st * (n - 1) + reach
        _pre(not _overlap(k, v), "k and v share memory", "alias", "v")
        for s, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if s is not None:
                _pre(codes, f"{name}: a bf16 cache has no scales", "argument", name)
                _check(s, name, torch.float32, 1, k.device, align=4)
                _dense(s, name)
                _pre(s.shape[0] == kv_heads, f"{name}: {s.shape[0]} of them for {kv_heads} heads", "shape", name)
        desc = N.PagedCacheDescriptor(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if k_scale is not None else None, v_scale.data_ptr() if v_scale is not None else None,
                                      pages, page_size, kv_heads, head_dim, strides[0], strides[1], strides[2], N.CACHE_E4M3 if codes else N.CACHE_BF16, 0)
        values = (k, v, k_scale, v_scale, pages, kv_heads, page_size, head_dim, k.device, k.get_device(), desc, ctypes.addressof(desc),
                  ((_span(k), "the cache's k"), (_span(v), "the cache's v")))
        for name, value in zip(PagedCache.__slots__, values, strict=True):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value) -> None:
        if name in PagedCache.__slots__:
            raise AttributeError(f"PagedCache.{name} cannot be exchanged: its tensors' contents may be changed in place, other tensors are another cache")
        object.__setattr__(self, name, value)

    def __reduce__(self):  # a copy is a cache over the tensors' copies
        return type(self), (self.k, self.v, self.k_scale, self.v_scale)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "bf16", *, k_scale=None, v_scale=None, device="cuda") -> "PagedCache":
        """A cache of its own memory, ``dtype`` "bf16" or "e4m3"; entries that were not written hold anything."""
        torch = _torch()
        _pre(dtype in ("bf16", "e4m3"), f"unknown cache dtype {dtype!r}", "dtype", "dtype")
        k, v = (torch.empty((pages, kv_heads, page_size, head_dim), dtype=torch.bfloat16 if dtype == "bf16" else torch.uint8, device=device) for _ in range(2))
        return cls(k, v, k_scale, v_scale)

    @property
    def dtype(self) -> str:
        return "bf16" if self._desc.dtype == N.CACHE_BF16 else "e4m3"

    def __repr__(self) -> str:
        return f"PagedCache({self.dtype}, pages={self.pages}, page_size={self.page_size}, kv_heads={self.kv_heads}, head_dim={self.head_dim})"


def _check_tables(tables, index: int):
    """(rows, columns, row stride, address) of int32 page tables."""
    torch = _torch()
    if not (isinstance(tables, torch.Tensor) and tables.dtype == torch.int32 and tables.dim() == 2 and tables.get_device() == index):
        _check(tables, "tables", torch.int32, 2, torch.device("cuda", index), align=4)
    rows, cols = tables.shape
    stride, inner = tables.stride()
    if cols == 0 or (inner != 1 and cols > 1):
        _pre(False, f"tables: rows must be dense and not empty (shape {tuple(tables.shape)})", "contiguous", "tables")
    return rows, cols, stride if rows > 1 else 0, tables.data_ptr()


def _check_cache(cache) -> None:
    if not isinstance(cache, PagedCache):
        _pre(False, f"cache: expected a PagedCache, got {type(cache).__name__}", "dtype", "cache")


def _heads(t, name: str, tokens: Optional[int], heads: Optional[int], dim: int, index: int):
    """``_rows`` of bf16 queries, keys, values or results of that many tokens and heads (None: any)."""
    got = _rows(t, name, _torch().bfloat16, index, 8, 16)
    shape = got[0]
    if (tokens is not None and shape[0] != tokens) or (heads is not None and shape[1] != heads) or shape[2] != dim:
        _pre(False, f"{name}: shape {tuple(shape)}, expected [{'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, {dim}]", "shape", name)
    return got


def cache_append(cache: PagedCache, k, v, tables, positions, *, rows=None, q=None, rotary: Optional[RotaryTable] = None, q_out=None, stream=None):
    """Writes the keys and values (bf16 [tokens, kv_heads, head_dim]) of new tokens into the cache, in one launch with the rotation of k and q.

    Token t becomes entry ``positions[t]`` (int32 or int64) of the sequence whose pages stand in row ``rows[t]`` of ``tables`` (int32 [sequences, width]);
    without ``rows`` the tokens belong to the sequences in turn, tokens / sequences each. With ``rotary`` k and q (bf16 [tokens, q_heads, head_dim]) are
    turned by ``positions``; returns the turned q (``q_out``, which may be q itself, or a new tensor), or None without q.

    k, v and q may lie in the cache's own memory (entries that move), but not in entries that this call writes: which ones those are stands on the device.

    A token with a negative position (padding), one beyond its table, a row outside the tables or a page outside the cache is not written. Where two
    tokens name one entry its content is unspecified: parts of both, or the key of one beside the value of the other. No entry of another position changes."""
    _check_cache(cache)
    index, dim = cache.index, cache.head_dim
    _here(index)
    kshape, kt, kh, kp = _heads(k, "k", None, cache.kv_heads, dim, index)
    tokens = kshape[0]
    krows, vrows = (kshape, kt, kh, kp), _heads(v, "v", tokens, cache.kv_heads, dim, index)
    _, vt, vh, vp = vrows
    seqs, cols, table_stride, tp = _check_tables(tables, index)
    pp, bits = _check_positions(positions, tokens, index)
    if rows is not None:
        rp = _ints(rows, "rows", tokens, index)
    else:
        rp = None
        if tokens and (seqs == 0 or tokens % seqs):
            _pre(False, f"k: {tokens} tokens cannot be dealt out evenly to {seqs} sequences; give rows", "divisible", "k")
    if rotary is not None:
        _check_table(rotary, dim, index)
        turns, rot, layout, magnitude = rotary.turns.data_ptr(), rotary.rot, rotary._layout, rotary.magnitude
    else:
        turns, rot, layout, magnitude = None, 0, 0, 1.0
    q_heads, qp, qt, qh, op, ot, oh = 0, None, 0, 0, None, 0, 0
    if q is not None:
        qshape, qt, qh, qp = _heads(q, "q", tokens, None, dim, index)
        q_heads = qshape[1]
        if q_out is None:
            q_out = _torch().empty_strided(qshape, (q_heads * dim, dim, 1), dtype=q.dtype, device=cache.device)
            ot, oh, op = q_heads * dim, dim, q_out.data_ptr()
        else:
            orows = _heads(q_out, "q_out", tokens, q_heads, dim, index)
            _, ot, oh, op = orows
            _result(q_out, "q_out")
            _pre((op == qp and ot == qt and oh == qh) or not _overlap(q_out, q), "q_out overlaps q without being q", "alias", "q_out")
            _pre((_columns(orows, krows, 2) or not _overlap(q_out, k)) and (_columns(orows, vrows, 2) or not _overlap(q_out, v)), "q_out overlaps k or v", "alias", "q_out")
            if tokens and q_heads:
                _apart(*_ends(orows, 2), "q_out", cache._spans)
        if q_heads == 0:
            qp = op = None
    elif q_out is not None:
        _pre(False, "q_out without q", "argument", "q_out")
    if tokens == 0:
        return q_out
    if seqs == 0:
        _pre(False, "tables: no sequences", "shape", "tables")
    N.check(N.load().tf_cache_append(cache._ref, kp, kt, kh, vp, vt, vh, tokens, tp, seqs, cols, table_stride, pp, bits, rp, qp, q_heads, qt, qh, op, ot, oh, turns, rot,
                                     layout, magnitude, _stream(stream)), "tf_cache_append")
    return q_out


# ---- attention over the cache ---------------------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device: int, seqs: int, queries: int, q_heads: int, kv_heads: int, dim: int, dtype: int, entries: int) -> int:
    return int(N.load().tf_paged_attention_workspace_bytes(seqs, queries, q_heads, kv_heads, dim, dtype, entries))


def paged_attention(q, cache: PagedCache, tables, lengths, *, counts=None, scale: Optional[float] = None, window: int = 0, out=None, return_lse: bool = False,
                    lse=None, workspace=None, stream=None):
    """Attention of the last tokens of each sequence over its entries in the cache; bf16 [tokens, q_heads, head_dim].

    ``q``        bf16 [sequences * queries, q_heads, head_dim]; q_heads a multiple of the cache's kv_heads (which share their queries' heads evenly)
    ``tables``   int32 [sequences, width]: the pages of each sequence; those behind its length are not looked at
    ``lengths``  int32 [sequences]: entries of each sequence, the new tokens' among them (``cache_append`` comes first)
    ``counts``   int32 [sequences]: how many of a sequence's queries are real (None: all); the others are padding at its end

    The last real query of a sequence sees all its entries, the one before all but the last, and so on; ``window`` > 0 bounds it to that many of the newest.
    ``scale`` is 1 / sqrt(head_dim) unless given. With ``return_lse`` (or ``lse``, float32 [tokens, q_heads]) returns (out, lse), lse = ln of the sum of
    exp(scale * q . k). A query that sees nothing (padding, an empty sequence) gets 0 and -inf. Entries on pages outside the cache are seen by nobody, and
    what is not seen does not matter, infinities and NaN included.

    f32 arithmetic, one rounding of the result, but for softmax weights, which are multiplied with the values in 16 bits (bf16 cache) or 11 (e4m3), and queries of
    an e4m3 cache, which are exact down to 2^-31 of their head's largest element."""
    torch = _torch()
    _check_cache(cache)
    index, dim, kv_heads = cache.index, cache.head_dim, cache.kv_heads
    _here(index)
    qrows = _heads(q, "q", None, None, dim, index)
    shape, qt, qh, qp = qrows
    tokens, heads = shape[0], shape[1]
    seqs, width, table_stride, tp = _check_tables(tables, index)
    lp = _ints(lengths, "lengths", seqs, index)
    cp = _ints(counts, "counts", seqs, index) if counts is not None else None
    if heads == 0 or heads % kv_heads:
        _pre(False, f"q: {heads} heads are not a multiple of the cache's {kv_heads}", "divisible", "q")
    if tokens and (seqs == 0 or tokens % seqs):
        _pre(False, f"q: {tokens} tokens cannot be dealt out evenly to {seqs} sequences", "divisible", "q")
    if scale is None:
        scale = dim**-0.5
    elif not abs(scale) <= 2.0**127:
        _pre(False, f"scale: {scale} is not a finite float32", "argument", "scale")
    if not (isinstance(window, int) and 0 <= window < 2**63):
        _pre(False, f"window: {window!r} is no whole number of 0 to 63 bits", "argument", "window")
    if out is None:
        out = torch.empty_strided(shape, (heads * dim, dim, 1), dtype=q.dtype, device=cache.device)
        ot, oh, op = heads * dim, dim, out.data_ptr()
    else:
        orows = _heads(out, "out", tokens, heads, dim, index)
        _, ot, oh, op = orows
        _result(out, "out")
        if tokens:
            (lo, hi), (first, end) = _ends(orows, 2), _ends(qrows, 2)
            if lo < end and first < hi:
                _pre(not _overlap(out, q), "out overlaps q", "alias", "out")
            _apart(lo, hi, "out", cache._spans)
    if lse is not None:
        _check(lse, "lse", torch.float32, 2, cache.device, align=4)
        _pre(tuple(lse.shape) == (tokens, heads), f"lse: shape {tuple(lse.shape)}, expected {(tokens, heads)}", "shape", "lse")
        _dense(lse, "lse")
        if tokens:
            _apart(*_span(lse), "lse", (*cache._spans, (_span(q), "q"), (_span(out), "out")))
        return_lse = True
    elif return_lse:
        lse = torch.empty_strided((tokens, heads), (heads, 1), dtype=torch.float32, device=cache.device)
    if tokens:
        queries = tokens // seqs
        need = _workspace_bytes(index, seqs, queries, heads, kv_heads, dim, cache._desc.dtype, width * cache.page_size)
        if need < 0:
            _pre(False, f"q: {seqs} sequences of {queries} queries are more than this operator takes", "unsupported", "q")
        if workspace is None:
            workspace, have = torch.empty(need, dtype=torch.uint8, device=cache.device), need
        else:
            _check(workspace, "workspace", torch.uint8, 1, cache.device)
            _dense(workspace, "workspace")
            have = workspace.numel()
            _pre(have >= need, f"workspace: {need} bytes needed", "workspace", "workspace")
            at = workspace.data_ptr()
            _apart(at, at + need, "workspace", (*cache._spans, (_ends(qrows, 2), "q"), (_ends((shape, ot, oh, op), 2), "out"), ((lp, lp + 4 * seqs), "lengths"),
                                                ((tp, tp + 4 * ((seqs - 1) * table_stride + width)), "tables")))
            if cp is not None:
                _apart(at, at + need, "workspace", (((cp, cp + 4 * seqs), "counts"),))
            if return_lse:
                _apart(at, at + need, "workspace", ((_span(lse), "lse"),))
        N.check(N.load().tf_paged_attention(cache._ref, qp, qt, qh, seqs, queries, heads, tp, width, table_stride, lp, cp, scale, window, op, ot, oh,
                                            lse.data_ptr() if return_lse else None, workspace.data_ptr(), have, _stream(stream)), "tf_paged_attention")
    return (out, lse) if return_lse else out


def attention_workspace_bytes(cache: PagedCache, sequences: int, queries: int, q_heads: int, width: int) -> int:
    """Bytes of the ``workspace`` that ``paged_attention`` takes for tables of ``width`` pages (for callers that keep one; it must not serve two calls at once)."""
    _check_cache(cache)
    _here(cache.index)  # the size goes by the current device's number of SMs
    need = _workspace_bytes(cache.index, sequences, queries, q_heads, cache.kv_heads, cache.head_dim, cache._desc.dtype, width * cache.page_size)
    if need < 0:
        _pre(False, f"paged_attention does not take {sequences} sequences of {queries} queries of {q_heads} heads over {cache.kv_heads}, tables of {width} pages", "unsupported")
    return need


# ---- the block ------------------------------------------------------------------------------------------------------------------


@dataclass
class AttentionWeights:
    """One layer's attention weights on one device. ``w_qkv``: [(q_heads + 2 kv_heads) * head_dim, H] (query, key, value rows); ``w_o``: [H, q_heads * head_dim]."""

    w_n: "object"  # bf16 [H]
    w_qkv: K.BlockScaledTensor
    w_o: K.BlockScaledTensor
    q_heads: int
    kv_heads: int

    @property
    def fmt(self) -> str:
        return self.w_qkv.fmt


def quantize_attention_weights(w_n, w_qkv, w_o, fmt: str, *, q_heads: int, kv_heads: int) -> AttentionWeights:
    """Quantizes bf16 ``w_qkv`` [(q_heads + 2 kv_heads) * head_dim, H] and ``w_o`` [H, q_heads * head_dim]."""
    rows, h = w_qkv.shape
    _pre(q_heads > 0 and kv_heads > 0 and q_heads % kv_heads == 0, f"q_heads={q_heads} is not a multiple of kv_heads={kv_heads}", "divisible", "q_heads")
    _pre(rows % (q_heads + 2 * kv_heads) == 0, f"w_qkv: {rows} rows are not {q_heads} + 2 * {kv_heads} heads", "shape", "w_qkv")
    dim = rows // (q_heads + 2 * kv_heads)
    _pre(tuple(w_o.shape) == (h, q_heads * dim), f"w_o: shape {tuple(w_o.shape)}, expected {(h, q_heads * dim)}", "shape", "w_o")
    return AttentionWeights(w_n, K.quantize(w_qkv, fmt), K.quantize(w_o, fmt), q_heads, kv_heads)


def _check_product(b, name: str, rows: int, k: int, device) -> None:
    if not (isinstance(b, K.BlockScaledTensor) and b.layout == "swizzled" and tuple(b.shape) == (rows, k) and b.device == device):
        _pre(isinstance(b, K.BlockScaledTensor) and b.layout == "swizzled", f"{name}: expected a BlockScaledTensor with swizzled scales", "dtype", name)
        _pre(tuple(b.shape) == (rows, k), f"{name}: shape {tuple(b.shape)}, expected {(rows, k)}", "shape", name)
        _pre(False, f"{name}: on {b.device}, the other arguments are on {device}", "device", name)


def _check_block(x, w, cache, tables, positions, lengths, rotary, rows, counts, window) -> None:
    """What the operators of ``attention_block`` would refuse, before the first of them has changed the residual or the cache."""
    _check_cache(cache)
    index, dim = cache.index, cache.head_dim
    _here(index)
    _check(x, "x", _torch().bfloat16, 2, cache.device)
    tokens, h = x.shape
    _pre(w.w_qkv.shape[0] == (w.q_heads + 2 * w.kv_heads) * dim and w.kv_heads == cache.kv_heads,
         f"the weights' heads ({w.q_heads} + 2 * {w.kv_heads}, {w.w_qkv.shape[0]} rows) do not match the cache's ({cache.kv_heads} of {dim})", "shape", "cache")
    _check_product(w.w_qkv, "w_qkv", w.w_qkv.shape[0], h, cache.device)
    _check_product(w.w_o, "w_o", h, w.q_heads * dim, cache.device)
    seqs = _check_tables(tables, index)[0]
    _check_positions(positions, tokens, index)
    if rows is not None:
        _ints(rows, "rows", tokens, index)
    if rotary is not None:
        _check_table(rotary, dim, index)
    _ints(lengths, "lengths", seqs, index)
    if counts is not None:
        _ints(counts, "counts", seqs, index)
    if tokens and (seqs == 0 or tokens % seqs):
        _pre(False, f"x: {tokens} tokens cannot be dealt out evenly to {seqs} sequences", "divisible", "x")
    if tokens and _workspace_bytes(index, seqs, tokens // seqs, w.q_heads, w.kv_heads, dim, cache._desc.dtype, tables.shape[1] * cache.page_size) < 0:
        _pre(False, f"x: {seqs} sequences of {tokens // seqs} tokens are more than paged_attention takes", "unsupported", "x")
    if not (isinstance(window, int) and 0 <= window < 2**63):
        _pre(False, f"window: {window!r} is no whole number of 0 to 63 bits", "argument", "window")


def attention_block(x, residual, w: AttentionWeights, cache: PagedCache, tables, positions, lengths, rotary: Optional[RotaryTable] = None, *, rows=None, counts=None,
                    window: int = 0, eps: float = 1e-6):
    """One attention block: ``residual += x`` (f32, in place), returns bf16 [tokens, H] = attention(rmsnorm(residual) * w_n) @ w_o^T, the keys and values of the
    tokens written into the cache on the way. ``positions``, ``tables``, ``rows`` as in ``cache_append``, ``lengths`` (after these tokens) and ``counts`` as in
    ``paged_attention``; the tokens of a sequence stand together, as many for each. A call that is refused has changed nothing."""
    torch = _torch()
    fmt = w.fmt
    _check_block(x, w, cache, tables, positions, lengths, rotary, rows, counts, window)
    tokens, dim = x.shape[0], cache.head_dim
    if fmt == "nvfp4":
        amax = torch.zeros(1, dtype=torch.float32, device=x.device)
        h = K.residual_add_rmsnorm(x, residual, w.w_n, eps, amax_out=amax)
        hq = K.quantize(h, fmt, amax=amax)
    else:
        _, hq = K.residual_add_rmsnorm(x, residual, w.w_n, eps, quantize_to=fmt, want_bf16=False)
    qkv = K.gemm_blockscaled(hq, w.w_qkv).view(tokens, w.q_heads + 2 * w.kv_heads, dim)
    q, k, v = qkv.split([w.q_heads, w.kv_heads, w.kv_heads], dim=1)
    cache_append(cache, k, v, tables, positions, rows=rows, q=q, rotary=rotary, q_out=q)
    o = paged_attention(q, cache, tables, lengths, counts=counts, window=window)
    return K.gemm(o.view(tokens, w.q_heads * dim), w.w_o)


def decoder_layer(x, residual, attention: AttentionWeights, mlp, cache: PagedCache, tables, positions, lengths, rotary: Optional[RotaryTable] = None, *, rows=None,
                  counts=None, window: int = 0, eps: float = 1e-6):
    """A whole decoder layer: ``attention_block``, then ``mlp.decoder_block`` on its result (``mlp``: ``MlpWeights``). The result is the next layer's ``x``."""
    from .mlp import decoder_block

    _check(x, "x", _torch().bfloat16, 2)
    _check_product(mlp.w_gu, "w_gu", 2 * mlp.w_d.shape[1], x.shape[1], x.device)
    _check_product(mlp.w_d, "w_d", x.shape[1], mlp.w_d.shape[1], x.device)
    _pre(mlp.w_gu.fmt == mlp.w_d.fmt, f"w_gu is {mlp.w_gu.fmt} but w_d is {mlp.w_d.fmt}", "dtype", "w_d")
    _check(mlp.w_n, "w_n", x.dtype, 1, x.device)
    _pre(mlp.w_n.shape[0] == x.shape[1], f"w_n: shape {tuple(mlp.w_n.shape)}, expected {(x.shape[1],)}", "shape", "w_n")
    y = attention_block(x, residual, attention, cache, tables, positions, lengths, rotary, rows=rows, counts=counts, window=window, eps=eps)
    return decoder_block(y, residual, mlp, eps)
