"""Low-rank adapters of many requests beside one projection.

The reference has no adapters; they stand beside its Linear (crates/theano-nn/src/linear.rs:111-121), whose
quantized weight all requests share:

    adapters = Adapters.from_tensors([(a0, b0), (a1, b1)], scales=[2.0, 0.5])
    y = linear(x, adapters, index)      # index: int32 [rows], each row's adapter, -1 for none
"""
from __future__ import annotations

import torch

from . import _abi
from ._tensor import stream
from .cache import _TYPES, _current_device, _dense, _device, _Fixed, _indices
from .errors import InvalidArgument

MAX_RANK = 256


class Adapters(_Fixed):
    """`count` adapters of a projection with K inputs and N outputs: y += scales[i] * b[i] @ (a[i] @ x).

    a: [count, rank, K], or [count, parts, rank, K] for a fused projection whose outputs are `parts`
    equal slices with adapters of their own (q, k and v); b: [count, N, rank]; bf16 or f16 device tensors,
    rank up to 256.  scales: float32 [count] or None (1).  Held are a copy of a in tiles of 16 ranks x 32 inputs (as the
    kernels load it, padded with zeros), scales themselves, and b itself, or a copy of it padded to ranks of 16 where it is not
    dense, of another rank or off 16 bytes: what is written to a afterwards changes nothing, what is written to scales or such a b
    changes the adapters."""

    def __init__(self, a, b, scales=None):
        a, b = _device(a, "Adapters: a").detach(), _device(b, "Adapters: b").detach()
        if a.dim() == 3:
            a = a.unsqueeze(1)
        if a.dtype not in (torch.bfloat16, torch.float16) or b.dtype != a.dtype or a.dim() != 4 or b.dim() != 3 or \
                b.shape[0] != a.shape[0] or b.shape[2] != a.shape[2] or not 1 <= a.shape[2] <= MAX_RANK or a.shape[0] < 1 or \
                not 1 <= a.shape[1] <= 16 or b.shape[1] % a.shape[1] or a.shape[3] < 1 or b.shape[1] < 1:
            raise InvalidArgument(f"Adapters: expected bfloat16 or float16 [count, (parts,) rank, K] and [count, N, rank], got "
                                  f"{a.dtype} {tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
        if scales is not None:
            _indices(scales, torch.float32, 1, "Adapters: scales")
            if scales.shape[0] != a.shape[0]:
                raise InvalidArgument(f"Adapters: {scales.shape[0]} scales for {a.shape[0]} adapters")
        count, parts, rank, k = a.shape
        n, row, ranks = b.shape[1], (k + 63) // 64 * 64, (rank + 15) // 16 * 16
        held = a.new_empty(count, parts * ranks // 16, row // 32, 16, 32)
        a = a.contiguous()
        _abi.call("tq_repack_adapters_tiled", a.data_ptr(), count * parts, rank, k, held.data_ptr(), stream())
        a = held
        if ranks != rank or not b.is_contiguous() or b.data_ptr() % 16:
            held = b.new_zeros(count, n, ranks)
            held[..., :rank] = b
            b = held
        self.__dict__.update(
            a=a, b=b, scales=scales, count=count, parts=parts, rank=rank, in_features=k, out_features=n, device_index=a.get_device(),
            _desc=_abi.adapters_desc(a.data_ptr(), b.data_ptr(), 0 if scales is None else scales.data_ptr(), count, parts, ranks,
                                     k, n, _TYPES[a.dtype]))

    @staticmethod
    def from_tensors(pairs, scales=None, dtype=torch.bfloat16):
        """Adapters of any ranks, from (a, b) pairs: a [rank, K] (or [parts, rank, K]) and b [N, rank], rounded to `dtype`;
        scales: a number for each."""
        pairs = [(a if a.dim() == 3 else a.unsqueeze(0), b) for a, b in pairs]
        if not pairs or any(a.dim() != 3 or b.dim() != 2 or a.shape[1] != b.shape[1] or
                            (a.shape[0], a.shape[2], b.shape[0]) != (pairs[0][0].shape[0], pairs[0][0].shape[2], pairs[0][1].shape[0])
                            for a, b in pairs):
            raise InvalidArgument("Adapters.from_tensors: expected pairs of [(parts,) rank, K] and [N, rank] with the same parts, K and N")
        dev = torch.device("cuda", torch.cuda.current_device())
        rank = (max(b.shape[1] for _, b in pairs) + 15) // 16 * 16
        parts, _, k = pairs[0][0].shape
        a = torch.zeros(len(pairs), parts, rank, k, dtype=dtype, device=dev)
        b = torch.zeros(len(pairs), pairs[0][1].shape[0], rank, dtype=dtype, device=dev)
        for i, (x, y) in enumerate(pairs):
            a[i, :, :x.shape[1]] = x
            b[i, :, :y.shape[1]] = y
        if scales is not None:
            scales = torch.as_tensor(scales, dtype=torch.float32).to(dev)
        return Adapters(a, b, scales)

    def _fits(self, index, rows, in_features, out_features, name):
        """These are adapters of such a projection, and `index` says those of so many rows, all on the current device."""
        if not isinstance(index, torch.Tensor) or tuple(index.shape) != (rows,) or self.in_features != in_features or \
                self.out_features != out_features:
            raise InvalidArgument(f"{name}: adapters of [{out_features}, {in_features}] take an index of {rows} rows")
        if self.device_index != _current_device():
            raise InvalidArgument(f"{name}: the adapters and the current device differ")
        _dense(index, torch.int32, 1, self.device_index) or _indices(index, torch.int32, 1, f"{name}: index")

    def add(self, x, index, y, out=None):
        """y [rows, N] (f32) with each row's share added: x [rows, K] f32, bf16 or f16; index int32 [rows], the row's adapter,
        or a number outside 0 .. count - 1 for none.  out: where the sums go (y itself, or a tensor that shares no memory with
        x, index and y), a new tensor if None."""
        dev, k, n = self.device_index, self.in_features, self.out_features
        if dev != _current_device():
            raise InvalidArgument("Adapters.add: the adapters and the current device differ")
        _dense(index, torch.int32, 1, dev) or _indices(index, torch.int32, 1, "Adapters.add: index")
        m = index.shape[0]
        code = _TYPES.get(x.dtype) if isinstance(x, torch.Tensor) else None
        if code is None or x.shape != (m, k):
            raise InvalidArgument(f"Adapters.add: x must be a float32, bfloat16 or float16 tensor [{m}, {k}]")
        if not _dense(x, x.dtype, 2, dev):
            x = _device(x, "Adapters.add: x").contiguous()
        if not (_dense(y, torch.float32, 2, dev) or _indices(y, torch.float32, 2, "Adapters.add: y").is_contiguous()) or y.shape != (m, n):
            raise InvalidArgument(f"Adapters.add: y must be contiguous float32 [{m}, {n}] on the current GPU")
        if out is None:
            out = torch.empty_like(y)
        elif out is not y and (not (_dense(out, torch.float32, 2, dev) or _indices(out, torch.float32, 2, "Adapters.add: out").is_contiguous()) or
                               out.shape != (m, n)):
            raise InvalidArgument(f"Adapters.add: out must be contiguous float32 [{m}, {n}] on the current GPU")
        nb = _abi.entry("tq_adapters_workspace_bytes")(self._desc, m)
        ws = y.new_empty(nb // 4) if nb > 0 else None
        _abi.call("tq_adapters_add", self._desc, x.data_ptr(), code, m, index.data_ptr(), y.data_ptr(), out.data_ptr(),
                  None if ws is None else ws.data_ptr(), nb, stream())
        return out
