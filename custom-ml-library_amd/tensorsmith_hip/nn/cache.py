"""Preallocated KV cache on a hip device (reference ``src/tensorsmith/nn/cache.py``).

Same API, validation order and storage layout as the reference: keys and
values live in ``[B, H_kv, capacity, D]`` device arrays, ``append`` writes the
slice ``[:, :, length:length+T]`` after checking every shape and the
capacity, ``get`` returns views of the active prefix, and the optional int8
mode stores symmetric per-token/head codes with one fp32 scale each
(``scale = max(max|x| / 127, 1e-8)``, ``q = round(x / scale)``, ``:73-77``),
dequantised on ``get`` (``:91-98``).  The views ``get`` returns feed the decode
kernel directly (no copy: the kernel takes the cache's strides).

On the hip device an int8 append is one fused kernel
(``tsattn_kv_append_int8``: row max, scale, rounding and both writes), and
``MultiHeadAttention`` decodes over the int8 storage itself
(``tsattn_decode_forward_int8`` dequantises inside the kernel) instead of
going through ``get``.
"""

from __future__ import annotations

import math
import operator

import numpy as np

import ctypes

from .. import _lib
from ..device import current_stream, launch
from .attention import _dtype_code, _rotate_at, _view, check_rotary, rope_tables
from ..device import device as parse_device
from ..tensor import Tensor, backend_dtype, is_grad_enabled, to_numpy


class KVCache:
    """Preallocated [B,H,capacity,D] keys/values for autoregressive inference."""

    def __init__(self, batch_size: int, num_heads: int, head_dim: int, max_seq_len: int, *,
                 device=None, dtype="float32", quantized: bool = False, value_dim=None):
        if min(batch_size, num_heads, head_dim, max_seq_len) <= 0:
            raise ValueError("cache dimensions and capacity must be positive")
        self.batch_size, self.num_heads, self.head_dim = batch_size, num_heads, head_dim
        self.value_dim = head_dim if value_dim is None else value_dim
        if self.value_dim <= 0:
            raise ValueError("value_dim must be positive")
        self.max_seq_len = max_seq_len
        self.device = parse_device(device)
        if self.device.type != "hip":
            raise RuntimeError("tensorsmith_hip keeps KV caches on hip devices")
        self.dtype = backend_dtype(dtype, self.device)
        if "float" not in str(self.dtype):
            raise TypeError("cache compute dtype must be floating point")
        self.quantized = quantized
        self.length = 0
        import torch

        dev = self.device.torch
        storage = torch.int8 if quantized else self.dtype
        shape = (batch_size, num_heads, max_seq_len)
        self._keys = torch.zeros(shape + (head_dim,), dtype=storage, device=dev)
        self._values = torch.zeros(shape + (self.value_dim,), dtype=storage, device=dev)
        self._key_scales = torch.ones(shape + (1,), dtype=torch.float32, device=dev) if quantized else None
        self._value_scales = (torch.ones(shape + (1,), dtype=torch.float32, device=dev)
                              if quantized else None)

    _described: tuple = ()

    def __getstate__(self):
        """What copies and pickles take: the views of ``_views`` are this cache's arrays' own."""
        return {name: value for name, value in self.__dict__.items() if name != "_described"}

    def append(self, key: Tensor, value: Tensor) -> tuple[Tensor, Tensor]:
        """Append a chunk after validating all shapes and capacity."""
        self._append(key, value)
        return self.get()

    def _append(self, key: Tensor, value: Tensor) -> None:
        """``append`` without building the returned views."""
        stop = self._check(key, value)
        window = slice(self.length, stop)
        keys, values = key._data.to(self.dtype), value._data.to(self.dtype)
        if self.quantized:
            _append_int8(keys, self._keys, self._key_scales, self.length, self.device)
            _append_int8(values, self._values, self._value_scales, self.length, self.device)
        else:
            self._keys[:, :, window] = keys
            self._values[:, :, window] = values
        self.length = stop

    def _append_rotary(self, key: Tensor, value: Tensor, base: float = 10000.0) -> bool:
        """Rotate ``key`` by RoPE at positions ``length ..`` and append it with
        ``value`` in one kernel (``tsattn_rope_append``).

        Same result as ``rotary_embedding(key, self.length)`` followed by
        ``_append``: the rotation runs in the key dtype, which must be the
        cache dtype here (else False is returned and nothing is written, so
        the caller takes the two-step path).  Needs an even head dim
        <= 512 equal to the value dim.
        """
        import torch

        if (key._data.dtype != self.dtype or value._data.dtype != self.dtype
                or self.dtype not in (torch.float32, torch.float16, torch.bfloat16)
                or self.head_dim % 2 or self.head_dim > 512 or self.value_dim != self.head_dim):
            return False
        stop = self._check(key, value)
        cos, sin = rope_tables(base, self.head_dim, self.dtype, self._keys.device, stop)
        k, v = key._data, value._data
        k = k if k.stride(-1) == 1 else k.contiguous()
        v = v if v.stride(-1) == 1 else v.contiguous()
        b, h, t, d = k.shape
        scales = ((ctypes.byref(_view(self._key_scales)), ctypes.byref(_view(self._value_scales)))
                  if self.quantized else (None, None))
        _lib.check(
            _lib.load().tsattn_rope_append(
                _CODES[str(k.dtype)], b, h, t, d, d, ctypes.byref(_view(k)), ctypes.byref(_view(v)),
                ctypes.byref(_view(self._keys)), ctypes.byref(_view(self._values)), *scales,
                ctypes.c_void_p(cos.data_ptr()), ctypes.c_void_p(sin.data_ptr()), self.length,
                ctypes.c_void_p(current_stream(self.device))),
            "RoPE cache append")
        self.length = stop
        return True

    def append_tree(self, key: Tensor, value: Tensor, tree, *, rotary_base: float | None = None) -> None:
        """Append the rows of drafted tokens [B, H, T, D] (``DraftTree``), the keys rotated by RoPE at their own
        positions, the cached length plus their depths, where ``rotary_base`` is given: one kernel
        (``tsattn_draft_append``)."""
        import torch

        stop = self._check(key, value)
        tree._check(self.batch_size, key.shape[2], self.device)
        check_rotary(rotary_base, self.head_dim)
        if (key._data.dtype != self.dtype or value._data.dtype != self.dtype
                or self.dtype not in (torch.float32, torch.float16, torch.bfloat16)
                or self.head_dim % 2 or self.head_dim > 512 or self.value_dim != self.head_dim):
            if rotary_base is not None:
                key = Tensor._leaf(_rotate_at(key._data, self.length + tree._depths, rotary_base), self.device)
            return self._append(key, value)
        cos = sin = None
        if rotary_base is not None:
            cos, sin = (x.data_ptr() for x in rope_tables(rotary_base, self.head_dim, self.dtype, self._keys.device, stop))
        k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (key._data, value._data))
        b, h, t, d = k.shape
        _lib.check(launch(self.device, _lib.load().tsattn_draft_append, _CODES[str(k.dtype)], b, h, t, d, _view(k),
                          _view(v), *self._views(), cos, sin, self.length, tree._depths.data_ptr(), tree.trees),
                   "draft append")
        self.length = stop

    def keep(self, first: int, index) -> None:
        """Of the positions from ``first`` on, keep those that ``index`` [B, n] names (n at most 256, counted from
        ``first``): they become the positions first .. first + n - 1, the cache's last.  One kernel reads all of them
        before it writes any (``tsattn_cache_keep``), so their order is free.  Indices on the host are checked; a hip
        tensor's are not waited for, and where one is out of range the position keeps what it held."""
        first = operator.index(first)
        if not 0 <= first <= self.length:
            raise ValueError("first must be between zero and the current length")
        drafted = self.length - first
        on_device = isinstance(index, Tensor) and index.device.type == "hip"
        if on_device and index.device != self.device:
            raise ValueError("kept indices must be on the cache's device")
        if not on_device:
            index = np.asarray(index.numpy() if isinstance(index, Tensor) else index)
        if "int" not in str(index.dtype) and 0 not in index.shape:
            raise TypeError("kept indices must have an integer dtype")
        if len(index.shape) != 2 or index.shape[0] != self.batch_size or index.shape[1] > min(drafted, 256):
            raise ValueError("kept indices must be [batch, positions], at most 256 and no more than there are")
        import torch

        if not on_device:
            if (index < 0).any() or (index >= drafted).any():
                raise ValueError("kept index out of range")
            index = Tensor._leaf(torch.from_numpy(index.astype(np.int64)).to(self._keys.device), self.device)
        n = index.shape[1]
        if n:
            raw = index._data if index._data.dtype in (torch.int64, torch.int32) else index._data.long()
            raw = raw.contiguous()
            _lib.check(launch(self.device, _lib.load().tsattn_cache_keep, self.batch_size, self.num_heads, n, first,
                              drafted, raw.data_ptr(), raw.element_size(), self._keys.element_size(), self.head_dim,
                              self.value_dim, *self._views()), "cache rows")
        self.length = first + n

    def _project_append(self, input: Tensor, projections, num_heads: int, rotary: bool,
                        base: float = 10000.0):
        """The cached attention step's q / k / v projections (``projections``:
        the q, k, v ``Linear`` layers), RoPE of q and k at positions
        ``length ..`` and the k / v append, in one kernel
        (``tsattn_qkv_rope_append``).  Returns the rotated queries [B, H, T, D]
        (a device tensor) and advances ``length``; or None, writing nothing,
        when the operands are outside the kernel (16-bit input in the cache
        dtype and the layers' dtype, head dim 64 / 128 equal to the value dim,
        embed a multiple of 16): the caller then projects and appends in steps.
        """
        import torch

        x = input._data
        lin = [(layer.weight._data, None if layer.bias is None else layer.bias._data)
               for layer in projections]
        tensors = [t for pair in lin for t in pair if t is not None]
        if (x.dtype != self.dtype or self.dtype not in (torch.float16, torch.bfloat16)
                or self.head_dim not in (64, 128) or self.value_dim != self.head_dim
                or x.ndim != 3 or x.shape[0] != self.batch_size or x.shape[-1] % 16
                or x.stride(-1) != 1 or x.data_ptr() % 16 or x.stride(0) % 8 or x.stride(1) % 8
                or any(t.dtype != x.dtype or not t.is_contiguous() or t.data_ptr() % 16
                       for t in tensors)
                or lin[0][0].shape[0] != num_heads * self.head_dim
                or any(w.shape[0] != self.num_heads * self.head_dim for w, _ in lin[1:])):
            return None
        b, t, e = x.shape
        stop = self.length + t
        if t == 0 or stop > self.max_seq_len:
            raise ValueError(f"cache capacity {self.max_seq_len} exceeded or empty append")
        q = torch.empty((b, num_heads, t, self.head_dim), dtype=x.dtype, device=x.device)
        cos = sin = None
        if rotary:
            cos, sin = rope_tables(base, self.head_dim, self.dtype, self._keys.device, stop)
        ptr = lambda z: None if z is None else ctypes.c_void_p(z.data_ptr())
        scales = ((ctypes.byref(_view(self._key_scales)), ctypes.byref(_view(self._value_scales)))
                  if self.quantized else (None, None))
        code = _CODES[str(x.dtype)]
        _lib.check(
            _lib.load().tsattn_qkv_rope_append(
                code, b, t, e, num_heads, self.num_heads, self.head_dim, ctypes.byref(_view(x.unsqueeze(1))),
                *(ptr(w) for w, _ in lin), *(ptr(bias) for _, bias in lin), ctypes.byref(_view(q)),
                ctypes.byref(_view(self._keys)), ctypes.byref(_view(self._values)), *scales,
                ptr(cos), ptr(sin), self.length, ctypes.c_void_p(current_stream(self.device))),
            "fused projection, RoPE and cache append")
        self.length = stop
        return q

    def _check(self, key: Tensor, value: Tensor) -> int:
        """Validate an append (reference order, cache.py:54-70); return the new length."""
        if key.device != self.device or value.device != self.device:
            raise ValueError("cache and key/value tensors must be on the same device")
        if is_grad_enabled() and (key.requires_grad or value.requires_grad):
            raise RuntimeError("KVCache is inference-only; use no_grad() for differentiable inputs")
        rows, others = key._data.shape, value._data.shape
        if len(rows) != 4 or rows[:2] != (self.batch_size, self.num_heads) or rows[3] != self.head_dim:
            raise ValueError("key shape does not match cache configuration")
        if others != (*rows[:3], self.value_dim):
            raise ValueError("value shape does not match cache configuration")
        stop = self.length + rows[2]
        if rows[2] == 0 or stop > self.max_seq_len:
            raise ValueError(f"cache capacity {self.max_seq_len} exceeded or empty append")
        return stop

    def get(self, last: int | None = None) -> tuple[Tensor, Tensor]:
        """Keys and values of the active prefix, or of its ``last`` positions."""
        last = None if last is None else operator.index(last)
        if last is not None and not 0 <= last <= self.length:
            raise ValueError("last must be between zero and the current length")
        first = 0 if last is None else self.length - last
        part = slice(first, self.length)
        if not self.quantized:
            return tuple(Tensor._leaf(x[:, :, part], self.device) for x in (self._keys, self._values))
        import torch

        b, h, _, d = self._keys.shape
        made = tuple(torch.empty((b, h, self.length - first, dim), dtype=self.dtype, device=self._keys.device)
                     for dim in (d, self.value_dim))
        try:
            if self.length > first:
                _lib.check(launch(self.device, _lib.load().tsattn_kv_read_int8, _dtype_code(self.dtype), b, h, first,
                                  self.length - first, d, self.value_dim, *self._views(), *(x.data_ptr() for x in made)),
                           "cached values")
        except NotImplementedError:  # (float64, or more rows than the kernel counts)
            for x, scale, out in zip(self.storage[:2], self.storage[2:], made):
                torch.mul(x[:, :, part], scale[:, :, part], out=out)
        return tuple(Tensor._leaf(x, self.device) for x in made)

    def reset(self) -> None:
        """Reuse the allocation; future appends overwrite old entries."""
        self.length = 0

    def truncate(self, length: int) -> None:
        if not 0 <= length <= self.length:
            raise ValueError("truncate length must be between zero and the current length")
        self.length = length

    def reorder(self, indices) -> None:
        """Reorder or duplicate batch rows for fixed-width beam search."""
        host = to_numpy(indices._data if isinstance(indices, Tensor) else indices)
        host = np.asarray(host)
        if host.shape != (self.batch_size,) or host.dtype.kind not in "iu":
            raise ValueError("beam indices must be one integer per cache batch row")
        if (host < 0).any() or (host >= self.batch_size).any():
            raise ValueError("beam index out of range")
        import torch

        order = torch.as_tensor(host.astype(np.int64), device=self._keys.device)
        self._described = ()  # (it would hold the old keys)
        self._keys, self._values = self._keys[order], self._values[order]
        if self.quantized:
            self._key_scales = self._key_scales[order]
            self._value_scales = self._value_scales[order]

    def _views(self) -> tuple:
        """The library's views of the arrays (which ``reorder`` replaces), the scales' None without them."""
        if not self._described or self._described[0] is not self._keys:
            self._described = (self._keys, tuple(None if x is None else _view(x) for x in self.storage))
        return self._described[1]

    @property
    def storage(self) -> tuple:
        """Raw persistent arrays."""
        return self._keys, self._values, self._key_scales, self._value_scales

    @property
    def memory_bytes(self) -> int:
        """Allocated persistent payload, excluding temporary dequantised arrays."""
        arrays = [self._keys, self._values]
        if self.quantized:
            arrays += [self._key_scales, self._value_scales]
        return sum(math.prod(a.shape) * a.element_size() for a in arrays)

    def __len__(self):
        return self.length

    def __repr__(self):
        return (f"KVCache(length={self.length}, capacity={self.max_seq_len}, "
                f"quantized={self.quantized}, device='{self.device}')")


_CODES = {"torch.float32": _lib.F32, "torch.float16": _lib.F16, "torch.bfloat16": _lib.BF16}


def _append_int8(rows, codes, scales, pos: int, dev) -> None:
    """Quantise rows [B, H, T, D] (cache dtype) into codes[:, :, pos:pos+T] and
    scales[:, :, pos:pos+T] with the fused append kernel."""
    if rows.stride(-1) != 1:
        rows = rows.contiguous()
    b, h, t, d = rows.shape
    _lib.check(
        _lib.load().tsattn_kv_append_int8(
            _CODES[str(rows.dtype)], b, h, t, d, ctypes.byref(_view(rows)),
            ctypes.byref(_view(codes)), ctypes.byref(_view(scales)), pos,
            ctypes.c_void_p(current_stream(dev))),
        "int8 cache append")
