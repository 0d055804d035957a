"""Serving state of a decoder layer on 8-bit keys and values: rotary positions, a paged
key/value cache that quantizes as it is written, and attention over it.

The reference's MultiheadAttention (crates/theano-nn/src/transformer.rs:9-162) knows
neither positions nor a cache, so these have no counterpart there; the cache's formats
are the per-row INT8 and FP8 (e4m3) ones of ``quantize_per_channel_i8`` and
``quantize_per_channel_fp8`` on each token's head.

    cache = KVCache.allocate(pages=512, page=64, heads=8, head_dim=128)
    rotary = Rotary.from_base(128, base=500000.0)
    new = KVBatch(table, lengths, tokens=1)        # lengths count the new tokens
    q = cache.write_rotary(q, k, v, rotary, new)   # q turned; k turned, coded and stored; v coded and stored
    o = cache.attention(q, new)

q, k and v are f32, bf16 or f16 device tensors [tokens, heads, head_dim] whose last
dimension is dense (slices of a fused projection's output are read in place), head_dim
up to 128.  Device data (positions, tables, lengths, offsets) is not read on the host:
what it says is checked on the device, see ``KVBatch``.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _abi
from ._abi import heads_desc as _heads_desc
from ._tensor import stream
from .errors import InvalidArgument
from .qconfig import QuantDType

MAX_HEAD_DIM = 128
_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # tq_dtype
_CODES = {torch.int8: 0, torch.uint8: 3}  # tq_qdtype


_current_device = torch._C._cuda_getDevice


def _device(t, name):
    """`t` lies on the current device: the call goes to that device's current stream."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.get_device() != _current_device():
        raise InvalidArgument(f"{name}: expected a tensor on the current GPU")
    return t


def _indices(t, dtype, dim, name):
    """`t` as a tensor of `dtype` with `dim` dimensions on the current device, its last one dense."""
    if _device(t, name).dtype != dtype or t.dim() != dim or (not t.is_contiguous() and t.stride(-1) != 1 and t.shape[-1] > 1):
        raise InvalidArgument(f"{name}: expected a dense {dim}-D {dtype} tensor, got {t.dtype} {tuple(t.shape)}")
    return t


def _dense(t, dtype, dim, device):
    """Whether `t` is a dense tensor of `dtype` with `dim` dimensions on `device`: what `_indices` asks for, found out faster (a
    decoding step's calls are bound by the host)."""
    return t.__class__ is torch.Tensor and t.dtype is dtype and t.dim() == dim and t.is_contiguous() and t.get_device() == device


def _heads(t, name, dtype=None, tokens=None, heads=None, dim=None):
    """(tensor, descriptor, dtype code) of a [tokens, heads, head_dim] tensor."""
    _device(t, name)
    code = _TYPES.get(t.dtype)
    if code is None or (dtype is not None and t.dtype != dtype):
        raise InvalidArgument(f"{name}: expected {dtype or 'float32, bfloat16 or float16'}, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[2] < 1 or (tokens is not None and shape[0] != tokens) or \
            (heads is not None and shape[1] != heads) or (dim is not None and shape[2] != dim):
        raise InvalidArgument(f"{name}: expected [{'tokens' if tokens is None else tokens}, "
                              f"{'heads' if heads is None else heads}, {'head_dim' if dim is None else dim}], "
                              f"got {tuple(shape)}")
    token, head, last = t.stride()
    if last != 1 and shape[2] > 1:
        t = t.contiguous()
        token, head, _ = t.stride()
    return t, _heads_desc(t.data_ptr(), shape[1], token, head), code


class _Fixed:
    """Attributes are set once, where the descriptor of the C calls is packed from them (`x.lengths += 1`, which writes
    into the tensor and sets the attribute to it again, is fine)."""

    def __setattr__(self, name, value):
        if value is not self.__dict__.get(name):
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: make another {type(self).__name__}")


@functools.lru_cache(maxsize=64)
def _packed_axes(axes):
    """The axes of planes as tq_rotary_axes takes them, and how many there are."""
    if any(x not in (0, 1, 2, 3) for x in axes):
        raise InvalidArgument(f"Rotary: axes are numbers from 0 to 3, got {axes}")
    words = [0, 0]
    for i, x in enumerate(axes):
        words[i // 32] |= int(x) << 2 * (i % 32)
    return tuple(words), max(map(int, axes), default=0) + 1


class Rotary(_Fixed):
    """Rotary positions: plane i of a head turns by position * frequencies[i].

    frequencies: float64 device tensor of rotary_dim / 2 angles per position; the first
    rotary_dim elements of a head turn, the others pass.  Plane i is elements (i, i +
    rotary_dim / 2), or (2 i, 2 i + 1) if `interleaved`.  Outputs are multiplied by `scale`.

    axes: for positions of several axes (time, height, width of an image's patches), the axis
    (0 to 3) of each plane, see `axes_in_blocks` and `axes_in_turn`; positions are then int64
    [axes, tokens], or [tokens] where all axes are the same (text)."""

    def __init__(self, frequencies, interleaved=False, scale=1.0, axes=None):
        _indices(frequencies, torch.float64, 1, "Rotary: frequencies")
        r, interleaved, scale = 2 * frequencies.shape[0], bool(interleaved), float(scale)
        planes, count = (0, 0), 0
        if axes is not None:
            axes = tuple(axes)
            if len(axes) != r // 2 or r > MAX_HEAD_DIM:
                raise InvalidArgument(f"Rotary: axes are {r // 2} numbers from 0 to 3, one for each plane, got {axes}")
            planes, count = _packed_axes(axes)
        self.__dict__.update(frequencies=frequencies, interleaved=interleaved, scale=scale, rotary_dim=r, axes=axes,
                             _planes=planes, _axes=count,
                             _desc=_abi.rotary_desc(frequencies.data_ptr(), r, interleaved, False, scale))

    @staticmethod
    def from_base(rotary_dim, base=10000.0, interleaved=False, scaling=None, factor=1.0, original_length=None,
                  fast_turns=32.0, slow_turns=1.0, scale=None, axes=None):
        """base^(-2 i / rotary_dim), for contexts `factor` times as long as trained on by
        `scaling`: "linear" (positions divided by factor), "ntk" (base * factor^(r / (r - 2)))
        or "yarn" (planes that turn fewer than `slow_turns` times over `original_length`
        divided by factor, those that turn more than `fast_turns` times kept, a ramp
        between; scale 0.1 ln(factor) + 1 unless given)."""
        r = int(rotary_dim)
        if r < 0 or r % 2 or not base > 0 or not factor > 0:
            raise InvalidArgument(f"Rotary.from_base: rotary_dim={rotary_dim}, base={base}, factor={factor}")
        if scaling == "ntk":
            if r <= 2:
                raise InvalidArgument("Rotary.from_base: ntk scaling needs rotary_dim > 2")
            base = base * factor ** (r / (r - 2))
        elif scaling not in (None, "linear", "yarn"):
            raise InvalidArgument(f"Rotary.from_base: unknown scaling {scaling!r}")
        f = float(base) ** (-torch.arange(0, r, 2, dtype=torch.float64) / max(r, 1))
        if scaling == "linear":
            f = f / factor
        elif scaling == "yarn":
            if not original_length or base == 1.0:
                raise InvalidArgument("Rotary.from_base: yarn scaling needs original_length and a base other than 1")

            def plane(turns):
                return r * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

            low, high = max(math.floor(plane(fast_turns)), 0), min(math.ceil(plane(slow_turns)), r - 1)
            ramp = ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
            f = f / factor * ramp + f * (1.0 - ramp)
            if scale is None:
                scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        return Rotary(f.to(torch.device("cuda", torch.cuda.current_device())), interleaved,
                      1.0 if scale is None else scale, axes)

    @staticmethod
    def axes_in_blocks(sizes):
        """`axes` where the first sizes[0] planes turn by axis 0, the next sizes[1] by axis 1, and so on."""
        return tuple(x for x, n in enumerate(sizes) for _ in range(n))

    @staticmethod
    def axes_in_turn(planes, axes):
        """`axes` where plane i turns by axis i % axes.  (Layouts that interleave sections of unequal sizes, whose last planes stay with
        one axis, are such a tuple written by hand.)"""
        return tuple(i % axes for i in range(planes))

    def _positions(self, positions, n, name):
        """The descriptor of the axes for positions [axes, n]; None for [n] (one axis, or all alike)."""
        if self.axes is None or not isinstance(positions, torch.Tensor) or positions.dim() != 2:
            _indices(positions, torch.int64, 1, f"{name}: positions")
            if positions.shape[0] != n:
                raise InvalidArgument(f"{name}: {positions.shape[0]} positions for {n} rows")
            return None
        _indices(positions, torch.int64, 2, f"{name}: positions")
        if positions.shape[0] < self._axes or positions.shape[1] != n:
            raise InvalidArgument(f"{name}: positions are [{self._axes}, {n}], got {tuple(positions.shape)}")
        return _abi.rotary_axes_desc(self._axes, positions.stride(0), *self._planes)

    def apply(self, q, k, positions, inverse=False):
        """(q, k) [tokens, heads, head_dim] turned to int64 `positions` [tokens] (or [axes, tokens]); k may be None.
        inverse: turned back (the transpose, which is the gradient's rotation)."""
        q, dq, code = _heads(q, "Rotary.apply: q")
        n, _, d = q.shape
        _device(self.frequencies, "Rotary: frequencies")
        axes = self._positions(positions, n, "Rotary.apply")
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = dk = ko_ptr = None
        if k is not None:
            k, dk, _ = _heads(k, "Rotary.apply: k", q.dtype, n, None, d)
            ko = torch.empty_like(k, memory_format=torch.contiguous_format)
            ko_ptr = ko.data_ptr()
        desc = self._desc
        if inverse:
            desc = _abi.rotary_desc(self.frequencies.data_ptr(), self.rotary_dim, self.interleaved, True, self.scale)
        if axes is None:
            _abi.call("tq_rotary_apply", desc, positions.data_ptr(), n, dq, dk, code, d, qo.data_ptr(), ko_ptr, stream())
        else:
            _abi.call("tq_rotary_apply_axes", desc, axes, positions.data_ptr(), n, dq, dk, code, d, qo.data_ptr(), ko_ptr,
                      stream())
        return qo, ko


class KVBatch(_Fixed):
    """Which tokens a call is about.

    table: int32 [batch, pages] pages of each sequence; lengths: int32 [batch] its tokens,
    those of the call among them (they are the last).  Rows are sequence after sequence,
    `tokens` each; or, with `offsets` (int32 [batch + 1], non-decreasing), rows
    offsets[b] .. offsets[b + 1] - 1 of `rows` in all, no sequence more than `tokens`.

    The device checks what it reads: a row with no place (before position 0, past the
    table, on a page outside the cache, before offsets[0], of a sequence with more than `tokens`
    rows or past `rows`) is not written and reads as zeros, a key with no place is
    seen by nobody, rows behind the last sequence are left as they were.  Positions that one call
    writes must not share a page's place."""

    def __init__(self, table, lengths, tokens=1, offsets=None, rows=None):
        _indices(table, torch.int32, 2, "KVBatch: table")
        _indices(lengths, torch.int32, 1, "KVBatch: lengths")
        batch = lengths.shape[0]
        if table.shape[0] != batch:
            raise InvalidArgument(f"KVBatch: {table.shape[0]} table rows for {batch} sequences")
        if offsets is None:
            if rows not in (None, batch * tokens):
                raise InvalidArgument(f"KVBatch: {rows} rows of {batch} sequences with {tokens} tokens each")
            rows = batch * tokens
        else:
            _indices(offsets, torch.int32, 1, "KVBatch: offsets")
            if offsets.shape[0] != batch + 1 or rows is None:
                raise InvalidArgument("KVBatch: offsets are [batch + 1], with `rows` rows in all")
        tokens, rows = int(tokens), int(rows)
        self.__dict__.update(
            table=table, lengths=lengths, offsets=offsets, batch=batch, tokens=tokens, rows=rows,
            device_index=table.get_device(),
            _desc=_abi.kv_batch_desc(table.data_ptr(), table.stride(0), table.shape[1], lengths.data_ptr(),
                                     0 if offsets is None else offsets.data_ptr(), batch, tokens, rows))


class KVCache(_Fixed):
    """A paged 8-bit cache of keys and values.

    k, v: int8 (INT8) or uint8 (FP8 e4m3 bit patterns) [pages, heads, page, row], row =
    head_dim rounded up to 32, zeros past head_dim; k_scale, v_scale: float32 [pages, heads,
    page].  page is a multiple of 16."""

    def __init__(self, k, k_scale, v, v_scale, head_dim):
        code = _CODES.get(k.dtype)
        shape = k.shape
        if code is None or v.dtype != k.dtype or k.dim() != 4 or v.shape != shape or \
                shape[3] != (head_dim + 31) // 32 * 32 or not 1 <= head_dim <= MAX_HEAD_DIM:
            raise InvalidArgument(f"KVCache: expected int8 or uint8 [pages, heads, page, row] for head_dim={head_dim}, "
                                  f"got {k.dtype} {tuple(shape)} and {v.dtype} {tuple(v.shape)}")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32 or k_scale.shape != shape[:3] or \
                v_scale.shape != shape[:3]:
            raise InvalidArgument(f"KVCache: expected float32 scales {tuple(shape[:3])}")
        for t in (k, k_scale, v, v_scale):
            if not _device(t, "KVCache").is_contiguous():
                raise InvalidArgument("KVCache: buffers must be contiguous")
        head_dim = int(head_dim)
        self.__dict__.update(
            k=k, k_scale=k_scale, v=v, v_scale=v_scale, pages=shape[0], heads=shape[1], page=shape[2], head_dim=head_dim,
            device=k.device, device_index=k.get_device(),
            _ref=_abi.kv_cache_desc(k.data_ptr(), k_scale.data_ptr(), v.data_ptr(), v_scale.data_ptr(), shape[0], shape[1],
                                    shape[2], head_dim, code))

    @staticmethod
    def allocate(pages, page, heads, head_dim, dtype=QuantDType.Int8):
        """An empty cache on the current device."""
        if dtype not in (QuantDType.Int8, QuantDType.FP8):
            raise InvalidArgument(f"KVCache.allocate: INT8 or FP8, not {dtype!r}")
        dev = torch.device("cuda", torch.cuda.current_device())
        shape = (pages, heads, page, (head_dim + 31) // 32 * 32)
        code = torch.int8 if dtype == QuantDType.Int8 else torch.uint8
        k, v = (torch.zeros(shape, dtype=code, device=dev) for _ in range(2))
        ks, vs = (torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
        return KVCache(k, ks, v, vs, head_dim)

    def _here(self, new):
        """Cache, batch and current device are one."""
        if self.device_index != new.device_index or self.device_index != _current_device():
            raise InvalidArgument("KVCache: the cache, the batch and the current device differ")
        return new._desc

    def write(self, k, v, new):
        """Quantizes k and v [rows, heads, head_dim] into the places of the batch's rows."""
        b = self._here(new)
        k, dk, code = _heads(k, "KVCache.write: k", None, new.rows, self.heads, self.head_dim)
        v, dv, _ = _heads(v, "KVCache.write: v", k.dtype, new.rows, self.heads, self.head_dim)
        _abi.call("tq_kv_write", self._ref, b, dk, dv, code, stream())

    def write_rotary(self, q, k, v, rotary, new, positions=None):
        """The same with q [rows, query heads, head_dim] and k turned first; returns q turned.
        positions: int64 [rows] (or [axes, rows]), or None for the rows' places in their sequences."""
        b = self._here(new)
        q, dq, code = _heads(q, "KVCache.write_rotary: q", None, new.rows, None, self.head_dim)
        k, dk, _ = _heads(k, "KVCache.write_rotary: k", q.dtype, new.rows, self.heads, self.head_dim)
        v, dv, _ = _heads(v, "KVCache.write_rotary: v", q.dtype, new.rows, self.heads, self.head_dim)
        _device(rotary.frequencies, "Rotary: frequencies")
        axes = None if positions is None else rotary._positions(positions, new.rows, "KVCache.write_rotary")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if axes is None:
            _abi.call("tq_kv_write_rotary", self._ref, b, rotary._desc,
                      None if positions is None else positions.data_ptr(), dq, dk,
                      dv, code, out.data_ptr(), stream())
        else:
            _abi.call("tq_kv_write_rotary_axes", self._ref, b, rotary._desc, axes, positions.data_ptr(), dq, dk, dv, code,
                      out.data_ptr(), stream())
        return out

    def read(self, new, dtype=torch.float32, out=None):
        """(k, v) [rows, heads, head_dim] of the batch's rows: code * scale, rounded to dtype.
        out: a pair of such tensors to read into."""
        b = self._here(new)
        code = _TYPES.get(dtype)
        if code is None:
            raise InvalidArgument(f"KVCache.read: expected float32, bfloat16 or float16, got {dtype}")
        shape = (new.rows, self.heads, self.head_dim)
        if out is None:
            k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        else:
            k, v = out
            for t in out:
                if _device(t, "KVCache.read: out").shape != shape or t.dtype != dtype or not t.is_contiguous():
                    raise InvalidArgument(f"KVCache.read: out must be contiguous {dtype} {shape}")
        _abi.call("tq_kv_read", self._ref, b, code, k.data_ptr(), v.data_ptr(), stream())
        return k, v

    def attention(self, q, new, tree=None, scale=None, out=None):
        """softmax(scale q k^T) v of q [rows, query heads, head_dim] (a multiple of the cache's
        heads) over the cache; scale 1 / sqrt(head_dim) unless given.  Row t of a sequence's
        new tokens sees the keys before the new tokens and new tokens up to its own, or, with
        `tree` (int32 [rows, words], see tree_mask), those whose bits are set.  A row that
        sees nothing gives zeros.  Returns [rows, query heads, head_dim] in q's dtype."""
        b = self._here(new)
        q, dq, code = _heads(q, "KVCache.attention: q", None, new.rows, None, self.head_dim)
        if q.shape[1] % self.heads:
            raise InvalidArgument(f"KVCache.attention: {q.shape[1]} query heads over {self.heads} key heads")
        words, tp = 0, None
        if tree is not None:
            _indices(tree, torch.int32, 2, "KVCache.attention: tree")
            if tree.shape[0] != new.rows or 32 * tree.shape[1] < new.tokens or not tree.is_contiguous():
                raise InvalidArgument(f"KVCache.attention: tree must be contiguous [{new.rows}, {(new.tokens + 31) // 32}], "
                                      f"got {tuple(tree.shape)}")
            words, tp = tree.shape[1], tree.data_ptr()
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif _device(out, "KVCache.attention: out").shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
            raise InvalidArgument(f"KVCache.attention: out must be contiguous {q.dtype} {tuple(q.shape)}")
        nb = _abi.entry("tq_kv_attention_workspace_bytes")(self._ref, b, q.shape[1])
        ws = q.new_empty(nb, dtype=torch.uint8) if nb > 0 else None
        _abi.call("tq_kv_attention", self._ref, b, dq, code, tp, words,
                  1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), None if ws is None else ws.data_ptr(),
                  nb, out.data_ptr(), stream())
        return out

    def keep(self, new, path, kept):
        """What of the new tokens was verified (see `verify_drafts`) stays: row path[b, i] of sequence b moves to
        the place of its i-th new token, for i < kept[b] (int32 [batch, n], ascending, and [batch]).  Returns the
        lengths that the sequences then have (int32 [batch]).  A sequence whose path does not ascend inside its rows stays
        as it is; one of whose kept rows lay nowhere (its page was missing) ends before the place that it would move to.  Pages that sequences share are copied first (PagePool.fork does)."""
        b, dev = self._here(new), self.device_index
        _dense(path, torch.int32, 2, dev) or _indices(path, torch.int32, 2, "KVCache.keep: path")
        _dense(kept, torch.int32, 1, dev) or _indices(kept, torch.int32, 1, "KVCache.keep: kept")
        if path.shape[0] != new.batch or kept.shape[0] != new.batch:
            raise InvalidArgument(f"KVCache.keep: paths {tuple(path.shape)} and kept {tuple(kept.shape)} of {new.batch} sequences")
        lengths = torch.empty_like(kept)
        _abi.call("tq_kv_keep", self._ref, b, path.data_ptr(), path.stride(0), path.shape[1], kept.data_ptr(),
                  lengths.data_ptr(), stream())
        return lengths

    def copy_pages(self, source, target):
        """Page target[j] becomes a copy of page source[j] (int32 [n] each, as PagePool.fork gives them; pairs with a page
        outside the cache are skipped).  A page is one pair's target and no pair's source."""
        dev = self.device_index
        _dense(source, torch.int32, 1, dev) or _indices(source, torch.int32, 1, "KVCache.copy_pages: source")
        _dense(target, torch.int32, 1, dev) or _indices(target, torch.int32, 1, "KVCache.copy_pages: target")
        if source.shape != target.shape or dev != _current_device():
            raise InvalidArgument(f"KVCache.copy_pages: {source.shape[0]} sources, {target.shape[0]} targets on the cache's device")
        _abi.call("tq_kv_copy_pages", self._ref, source.data_ptr(), target.data_ptr(), source.shape[0], stream())


def tree_mask(seen):
    """Bit words (int32 [rows, ceil(T / 32)], on `seen`'s device) of a bool tensor [rows, T]:
    bit j of a row is set where the row sees new token j of its sequence."""
    if seen.dtype != torch.bool or seen.dim() != 2:
        raise InvalidArgument("tree_mask: expected a bool [rows, T] tensor")
    rows, t = seen.shape
    words = max((t + 31) // 32, 1)
    bits = torch.zeros(rows, words * 32, dtype=torch.int64, device=seen.device)
    bits[:, :t] = seen
    v = (bits.view(rows, words, 32) << torch.arange(32, device=seen.device)).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).to(torch.int32)
