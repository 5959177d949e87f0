"""Attention of new tokens over a ``KVCache`` that they do not all see alike: drafted
tokens that form a tree, or a sliding window with sinks (the reference decodes token by
token over the whole cache, ``src/tensorsmith/nn/transformer.py:355-402``).

A round of drafted tokens: ``cache.append_tree(k, v, tree)`` puts them behind the cached
positions, ``cached_attention(q, cache, tree)`` lets each see those, its ancestors and
itself, and ``cache.keep(first, path)`` keeps an accepted path of them.
``MultiHeadAttention`` and ``TransformerLM`` do the first two for ``tree=``.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np

from .. import _lib
from ..device import device as parse_device
from ..device import launch, require_available
from ..tensor import Tensor, is_grad_enabled
from .attention import (_check_window, _dtype_code, _operand, _rotate_at, _view, check_rotary, rope_tables,
                        rotary_embedding, scaled_dot_product_attention)
from .cache import KVCache

__all__ = ["DraftTree", "cached_attention"]

MOST_TOKENS = 256


class DraftTree:
    """Drafted tokens as a tree, for all sequences of a batch or one for each.

    ``parents`` [T] or [B, T], T at most 256: each token's parent, an earlier token of its tree, or -1 for the last
    cached token.  Parents on the host are checked; a hip tensor's are not waited for, and one that is not an earlier
    token counts as -1.  A token's position is the cached length plus its depth (``depths`` [T] or [B, T]).
    """

    def __init__(self, parents, device=None):
        import torch

        on_device = isinstance(parents, Tensor) and parents.device.type == "hip"
        shape = tuple(parents.shape) if on_device else None
        if on_device:
            if device is not None and parse_device(device) != parents.device:
                raise ValueError("the tree's device is its parents'")
            if "int" not in str(parents.dtype):
                raise TypeError("parents must have an integer dtype")
        else:
            host = np.asarray(parents.numpy() if isinstance(parents, Tensor) else parents)
            if host.dtype.kind not in "iu" and host.size:
                raise TypeError("parents must have an integer dtype")
            shape = host.shape
        if len(shape) not in (1, 2) or 0 in shape or shape[-1] > MOST_TOKENS:
            raise ValueError(f"parents must be [tokens] or [batch, tokens], of 1 to {MOST_TOKENS} tokens")
        if not on_device and ((host < -1) | (host >= np.arange(shape[-1]))).any():
            raise ValueError("a token's parent is an earlier token, or -1")
        self.device = parents.device if on_device else require_available("hip" if device is None else device)
        if self.device.type != "hip":
            raise RuntimeError("tensorsmith_hip keeps draft trees on hip devices")
        self.tokens, self.trees, self._shape = shape[-1], shape[0] if len(shape) == 2 else 1, shape
        raw = parents._data if on_device else torch.from_numpy(host.astype(np.int32)).to(self.device.torch)
        if raw.dtype == torch.int64:  # (no value wraps round to an earlier token)
            raw = raw.clamp(-1, MOST_TOKENS)
        raw = raw.to(torch.int32).reshape(self.trees, self.tokens).contiguous()
        self._words = torch.empty((self.trees, self.tokens, -(-self.tokens // 32)), dtype=torch.int32, device=raw.device)
        self._depths = torch.empty((self.trees, self.tokens), dtype=torch.int32, device=raw.device)
        _lib.check(launch(self.device, _lib.load().tsattn_draft_tree, self.trees, self.tokens, raw.data_ptr(),
                          self._words.data_ptr(), self._depths.data_ptr()), "draft tree")

    @property
    def depths(self) -> Tensor:
        return Tensor._leaf(self._depths.reshape(self._shape), self.device)

    def _visible(self):
        """[trees, T, T]: whether token s is t or one of its ancestors."""
        import torch

        s = torch.arange(self.tokens, device=self._words.device)
        return (self._words[..., s // 32] >> (s % 32).to(torch.int32)) & 1 != 0

    def _check(self, batch: int, tokens: int, dev) -> None:
        if tokens != self.tokens or self.trees not in (1, batch):
            raise ValueError("the tree does not match the drafted tokens")
        if dev is not self.device and dev != self.device:
            raise ValueError("the tree must be on the device of its tokens")

    def __repr__(self):
        return f"DraftTree(tokens={self.tokens}, trees={self.trees}, device='{self.device}')"


def cached_attention(query: Tensor, cache: KVCache, tree: DraftTree | None = None, *, scale: float | None = None,
                     window: int | None = None, sinks: int = 0, rotary_base: float | None = None) -> Tensor:
    """Inference attention of ``query`` [B, Hq, T, D] over ``cache``, whose last T positions are the queries' own.

    Causal; through a ``window`` (and ``sinks``) as in ``scaled_dot_product_attention``, or with a ``tree`` of drafted
    tokens, each of which sees the positions in front of them (a window's, at its own position), its ancestors and
    itself.  ``rotary_base``: the queries are rotated by RoPE at their positions.  One kernel reads the cache's visible
    part once, int8 caches in int8 (``tsattn_cached_attend``); other dtypes and head dims, and more than 256 tokens, go
    through ``scaled_dot_product_attention``.  Cached values are taken to be finite: what a token does not see may share
    a tile with what it does."""
    if not isinstance(cache, KVCache):
        raise TypeError("cached_attention reads a KVCache")
    q, dev = query._data, query.device
    if len(q.shape) != 4:
        raise ValueError("attention expects [batch, heads, sequence, channels]")
    if dev is not cache.device and dev != cache.device:
        raise ValueError("attention tensors must be on the same device")
    if q.dtype != cache.dtype:
        raise TypeError("the queries must have the cache's dtype")
    if query.requires_grad and is_grad_enabled():
        raise RuntimeError("cached attention is inference-only; use no_grad() for differentiable inputs")
    b, heads, tokens, dim = q.shape
    if b != cache.batch_size or dim != cache.head_dim or heads == 0 or heads % cache.num_heads:
        raise ValueError("query shape does not match cache configuration")
    length = cache.length
    if not 0 < tokens <= length:
        raise ValueError("the queries' own positions must be in the cache")
    if scale is not None and not math.isfinite(scale):
        raise ValueError("attention scale must be finite")
    check_rotary(rotary_base, dim)
    whole = window
    window, sinks = _check_window(window, sinks, True, length)
    if tree is not None:
        tree._check(b, tokens, dev)
        if whole is not None and whole < tokens:
            raise ValueError("the window must hold the drafted tokens")
    import torch

    q, code = _operand(q), _dtype_code(q.dtype)
    if cache.value_dim == dim and code != _lib.F64:
        cos = sin = words = depths = ws = None
        trees = 0
        if tree is not None:
            trees, words, depths = tree.trees, tree._words.data_ptr(), tree._depths.data_ptr()
        if rotary_base is not None:
            cos, sin = (x.data_ptr() for x in rope_tables(rotary_base, dim, q.dtype, q.device, length))
        desc = _lib.Cached(code, b, heads, cache.num_heads, dim, tokens, length, cache.quantized,
                           1 / math.sqrt(dim) if scale is None else scale, window or 0, sinks, trees,
                           words, depths, cos, sin)
        lib = _lib.load()
        out = torch.empty((b, heads, tokens, dim), dtype=q.dtype, device=q.device)
        nbytes = lib.tsattn_cached_attend_workspace(desc)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        try:
            _lib.check(launch(dev, lib.tsattn_cached_attend, desc, _view(q), *cache._views(), _view(out),
                              None if ws is None else ws.data_ptr(), nbytes), "cached attention")
            return Tensor._leaf(out, dev)
        except NotImplementedError:  # outside the kernel
            pass
    first = length - tokens
    k, v = cache.get()
    if tree is None:
        q = query if rotary_base is None else rotary_embedding(query, first, rotary_base)
        return scaled_dot_product_attention(q, k, v, None, 0.0, True, scale=scale, causal_offset=first,
                                            enable_gqa=True, window=window, sinks=sinks)
    positions = first + tree._depths
    if rotary_base is not None:
        query = Tensor._leaf(_rotate_at(q, positions, rotary_base), query.device)
    j = torch.arange(first, device=q.device)
    past = torch.ones((tree.trees, tokens, first), dtype=torch.bool, device=q.device)
    if window is not None:
        past = (j > positions[..., None] - window) | (j < sinks)
    mask = Tensor._leaf(torch.cat((past, tree._visible()), -1)[:, None], query.device)
    return scaled_dot_product_attention(query, k, v, mask, 0.0, False, scale=scale, enable_gqa=True)
