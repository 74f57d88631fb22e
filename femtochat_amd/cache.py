"""Text generation on the MI355X: a cache of keys and values, and attention of the
newest tokens over it.

They stand beside ``attention`` for what follows training: a prompt's keys and
values (after the attention prologue) are written once, and each new token, or tree
of drafted ones, attends to them with the scores that ``attention`` gives (causal or
windowed, capped, biased).  The reference has no counterpart.

A ``KVCache`` holds tokens in pages::

    k, v              (pages, Hkv, page, D), bfloat16, int8 or float8_e4m3fn
    k_scale, v_scale  (pages, Hkv, page) float32, one per token and head (8-bit types)
    pages             (B, M) int32: the pages of each sequence's tokens in order, or
                      None, where page b is sequence b's own

or, with a leading dimension, those of all layers (``cache.layer(i)`` is one).  An
8-bit value is code * scale, with scale = max |x| / 127 (int8) or / 448 (float8) over a
token's head.  ``lengths`` (B,) int32 are the tokens that the cache holds before a
call; the call's own tokens lie behind them, ``counts`` (B,) int32 of them where a
batch is ragged.  None of the calls has a gradient.  A step of generation with drafted
tokens is::

    for i in range(layers):                       # nodes: the last token and the drafts
        cache_write_(cache.layer(i), K, V, lengths, counts)
        O = cached_attention(Q, cache.layer(i), lengths, window, parents=parents, counts=counts)
    path, kept, token = verify_drafts(logits, nodes, uniforms, parents=parents, counts=counts)
    cache_keep_(cache, lengths, path, kept)
    lengths += kept                               # token is the next step's first node
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .kernels import _call, _check_tensor, _check_workspace, _dtype_code, _ptr

__all__ = [
    "KVCache",
    "kv_cache",
    "cache_write_",
    "cache_read",
    "cache_read_",
    "cache_keep_",
    "cached_attention",
    "cached_attention_",
    "cached_attention_workspace_bytes",
]

_TYPES = {torch.bfloat16: _lib.FC_CACHE_BF16, torch.int8: _lib.FC_CACHE_I8, torch.float8_e4m3fn: _lib.FC_CACHE_F8}
_VALUES = (torch.float32, torch.bfloat16)
_I32 = (torch.int32,)
_F32 = (torch.float32,)
_BF16 = (torch.bfloat16,)


class KVCache(NamedTuple):
    """A cache's buffers (module documentation)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None
    pages: Optional[torch.Tensor] = None

    def layer(self, i: int) -> "KVCache":
        """Layer i of a cache of several."""
        if self.k.dim() != 5:
            raise ValueError("the cache holds one layer")
        pick = lambda t: None if t is None else t[i]  # noqa: E731
        return KVCache(self.k[i], self.v[i], pick(self.k_scale), pick(self.v_scale), self.pages)

    @property
    def capacity(self) -> int:
        """The tokens a sequence has room for."""
        return self.k.shape[-2] * (1 if self.pages is None else self.pages.shape[1])


def kv_cache(sequences: int, capacity: int, n_kv_head: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, *,
             layers: Optional[int] = None, page: Optional[int] = None, pool: Optional[int] = None, device="cuda") -> KVCache:
    """An empty cache for ``sequences`` of up to ``capacity`` tokens (rounded up to whole
    pages, of 16 tokens at least).  With ``page`` (a power of two from 16) it is a pool of ``pool``
    pages (default: enough for every sequence) and a table, filled in order as far as the
    pool goes and with -1 behind it; the caller may hand out pages otherwise."""
    if dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {dtype}; a cache holds bfloat16, int8 or float8_e4m3fn")
    if min(sequences, capacity, n_kv_head, head_dim) <= 0 or (layers is not None and layers <= 0) or (pool is not None and pool <= 0):
        raise ValueError("sequences, capacity, n_kv_head, head_dim, layers and pool must be positive")
    table = None
    if page is None:
        if pool is not None:
            raise ValueError("a pool has pages")
        size, count = -(-capacity // 16) * 16, sequences
    else:
        if page < 16 or page & (page - 1):
            raise ValueError("a page holds a power of two of tokens, 16 at least")
        each = -(-capacity // page)
        size, count = page, sequences * each if pool is None else pool
        table = torch.arange(sequences * each, dtype=torch.int32)
        table = torch.where(table < count, table, -1).view(sequences, each).to(device)
    shape = ((layers,) if layers is not None else ()) + (count, n_kv_head, size)
    k, v = (torch.zeros(shape + (head_dim,), dtype=dtype, device=device) for _ in range(2))
    if dtype == torch.bfloat16:
        return KVCache(k, v, None, None, table)
    return KVCache(k, v, torch.zeros(shape, device=device), torch.zeros(shape, device=device), table)


class _Layout:
    """What follows from a cache's shapes alone, once for each of them: a call on a few
    tokens is shorter than its preparation."""

    __slots__ = ("desc", "ref", "shape", "scales", "pages", "lead", "batch", "B", "Hkv", "D", "types", "bytes")

    def __init__(self, shape, dtype, pages, B: int):
        if len(shape) not in (4, 5) or dtype not in _TYPES:
            raise ValueError("a cache's k must be a ([layers,] pages, Hkv, page, D) tensor of bfloat16, int8 or float8_e4m3fn")
        if pages is not None and (len(pages) != 2 or pages[1] == 0):
            raise ValueError("a cache's pages must be a (B, M) int32 tensor")
        self.shape, self.types, self.lead, self.B = shape, (dtype,), tuple(shape[:-4]), B
        self.scales = None if dtype is torch.bfloat16 else shape[:-1]
        self.batch = (B,)
        self.pages = None if pages is None else (B, pages[1])
        P, self.Hkv, S, self.D = shape[-4:]
        self.desc = _lib.CacheDesc(self.D, self.Hkv, B, self.lead[0] if self.lead else 1, P, S, 0 if pages is None else pages[1], _TYPES[dtype])
        self.ref = ctypes.byref(self.desc)
        self.bytes = {}  # of attention's workspace, by what a call adds


_layout = lru_cache(maxsize=256)(_Layout)


class _Buffers(NamedTuple):
    """A checked cache: its layout, pointers and device."""

    layout: _Layout
    pointers: _lib.Cache
    device: torch.device


def _buffers(cache: KVCache, B: int) -> _Buffers:
    k, v, ks, vs, pages = cache
    if not isinstance(k, torch.Tensor):
        raise ValueError("a cache's k must be a ([layers,] pages, Hkv, page, D) tensor of bfloat16, int8 or float8_e4m3fn")
    if pages is not None and not isinstance(pages, torch.Tensor):
        raise ValueError("a cache's pages must be a (B, M) int32 tensor")
    layout = _layout(k.shape, k.dtype, None if pages is None else pages.shape, B)
    device = k.device
    if device.type != "cuda":
        raise ValueError("the MI355X cache kernels need tensors on a HIP device (torch 'cuda'); there is no CPU path")
    if not (k.is_contiguous() and isinstance(v, torch.Tensor) and v.shape == layout.shape and v.dtype is layout.types[0]
            and v.device == device and v.is_contiguous()):
        _check_tensor("k", k, layout.shape, layout.types, device)
        _check_tensor("v", v, layout.shape, layout.types, device)
    k_scale = v_scale = table = None
    if layout.scales is not None:
        if not (isinstance(ks, torch.Tensor) and isinstance(vs, torch.Tensor) and ks.shape == layout.scales and vs.shape == layout.scales
                and ks.dtype is torch.float32 and vs.dtype is torch.float32 and ks.device == device and vs.device == device
                and ks.is_contiguous() and vs.is_contiguous()):
            _check_tensor("k_scale", ks, layout.scales, _F32, device)
            _check_tensor("v_scale", vs, layout.scales, _F32, device)
        k_scale, v_scale = ks.data_ptr(), vs.data_ptr()
    elif ks is not None or vs is not None:
        raise ValueError("a bfloat16 cache has no scales")
    if pages is not None:
        _check_tensor("pages", pages, layout.pages, _I32, device)
        table = pages.data_ptr()
    return _Buffers(layout, _lib.Cache(k.data_ptr(), v.data_ptr(), k_scale, v_scale, table), device)


def _batch(cache: KVCache, like) -> int:
    """The sequences of a call: those of ``like`` (B, ...), or of the cache's table."""
    if isinstance(like, torch.Tensor) and like.dim() >= 1:
        return like.shape[0]
    rows = cache.k if cache.pages is None else cache.pages
    at = -4 if cache.pages is None else 0
    if not isinstance(rows, torch.Tensor) or rows.dim() < (4 if cache.pages is None else 1):
        raise ValueError("a cache is ([layers,] pages, Hkv, page, D) tensors and a (B, M) int32 table, or None for it")
    return rows.shape[at]


def _check_counts(c: _Buffers, lengths, counts, name: str = "lengths", required: bool = False) -> None:
    B, device = c.layout.batch, c.device
    if (lengths is not None or required) and not (isinstance(lengths, torch.Tensor) and lengths.shape == B and lengths.dtype is torch.int32
                                                  and lengths.device == device and lengths.is_contiguous()):
        _check_tensor(name, lengths, B, _I32, device)
    if counts is not None:
        _check_tensor("counts", counts, B, _I32, device)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """An input as the kernels read it, 16 bytes at a time."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def cache_write_(cache: KVCache, K: torch.Tensor, V: torch.Tensor, lengths: torch.Tensor,
                 counts: Optional[torch.Tensor] = None) -> None:
    """Writes K and V ([layers,] B, T, Hkv, D), float32 or bfloat16, as each sequence's
    tokens ``lengths[b]`` to ``lengths[b] + counts[b] - 1`` (T of them without ``counts``),
    quantised to the cache's type.  Tokens beyond the capacity are not written; ``lengths``
    is the caller's to move on, once all layers are written."""
    c = _buffers(cache, _batch(cache, lengths))
    T = _check_values(c, K, V)
    _check_counts(c, lengths, counts, required=True)
    if T == 0:
        return
    K, V = _aligned(K), _aligned(V)
    _call(c.device, _lib.lib().fc_cache_write, c.layout.ref, ctypes.byref(c.pointers), K.data_ptr(), V.data_ptr(),
          _dtype_code(K.dtype), T, lengths.data_ptr(), _ptr(counts))


def _check_values(c: _Buffers, K, V) -> int:
    layout, device = c.layout, c.device
    if not isinstance(K, torch.Tensor) or K.dim() != len(layout.shape):
        raise ValueError("K and V must be ([layers,] B, T, Hkv, D) tensors, with layers where the cache has them")
    shape = K.shape
    T = shape[-3]
    want = layout.lead + (layout.B, T, layout.Hkv, layout.D)
    if not (shape == want and K.dtype in _VALUES and K.device == device and K.is_contiguous() and isinstance(V, torch.Tensor)
            and V.shape == shape and V.dtype is K.dtype and V.device == device and V.is_contiguous()):
        _check_tensor("K", K, want, _VALUES, device)
        _check_tensor("V", V, want, (K.dtype,), device)
    return T


def cache_read_(K: torch.Tensor, V: torch.Tensor, cache: KVCache, starts: Optional[torch.Tensor] = None,
                counts: Optional[torch.Tensor] = None) -> None:
    """``cache_read`` into the caller's K and V."""
    c = _buffers(cache, _batch(cache, starts if starts is not None else counts))
    _check_values(c, K, V)
    if K.shape[-3] != 0 and (K.data_ptr() | V.data_ptr()) % 16:
        raise ValueError("K and V must start on a 16-byte boundary")
    _read(c, K, V, starts, counts)


def _read(c: _Buffers, K, V, starts, counts) -> None:
    _check_counts(c, starts, counts, "starts")
    T = K.shape[-3]
    if T == 0:
        return
    _call(c.device, _lib.lib().fc_cache_read, c.layout.ref, ctypes.byref(c.pointers), K.data_ptr(), V.data_ptr(),
          _dtype_code(K.dtype), T, _ptr(starts), _ptr(counts))


def cache_read(cache: KVCache, starts: Optional[torch.Tensor], T: int, counts: Optional[torch.Tensor] = None, *,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values ([layers,] B, T, Hkv, D) of each sequence's tokens ``starts[b]`` (None:
    0) to ``starts[b] + counts[b] - 1``, with zeros behind them, in float32 or bfloat16:
    ``cache_read(cache, None, T, lengths)`` is all that the cache holds, for ``attention``.
    Tokens beyond the capacity read as NaN."""
    if dtype not in _VALUES:
        raise TypeError(f"unsupported dtype {dtype}; a cache reads back as float32 or bfloat16")
    if T < 0:
        raise ValueError("T must not be negative")
    c = _buffers(cache, _batch(cache, starts if starts is not None else counts))
    layout = c.layout
    K = torch.empty(*layout.lead, layout.B, T, layout.Hkv, layout.D, dtype=dtype, device=c.device)
    V = torch.empty_like(K)
    _read(c, K, V, starts, counts)
    return K, V


def cache_keep_(cache: KVCache, lengths: torch.Tensor, path: torch.Tensor, counts: torch.Tensor) -> None:
    """Keeps a path of the tokens behind ``lengths``: token ``lengths[b] + path[b, j]`` moves to
    ``lengths[b] + j`` for j < counts[b], in every layer that the cache holds.  ``path`` (B, N)
    int32 increases along a row, as ``verify_drafts`` gives it."""
    c = _buffers(cache, _batch(cache, lengths))
    if not isinstance(path, torch.Tensor) or path.dim() != 2:
        raise ValueError("path must be a (B, N) int32 tensor")
    N = path.shape[1]
    B = c.layout.B
    _check_tensor("path", path, (B, N), _I32, c.device)
    _check_tensor("counts", counts, (B,), _I32, c.device)
    _check_counts(c, lengths, None, required=True)
    if N == 0:
        return
    _call(c.device, _lib.lib().fc_cache_keep, c.layout.ref, ctypes.byref(c.pointers), N, lengths.data_ptr(),
          path.data_ptr(), counts.data_ptr())


def _left(window) -> int:
    left, right = window
    if int(right) != 0 or int(left) < -1:
        raise ValueError(f"a window over a cache is (left, 0), or (-1, 0) for all tokens, got {tuple(window)}")
    return int(left)


def _options(c: _Buffers, N: int, H: int, window, parents, softcap, slopes) -> _lib.CachedAttnOptions:
    tree = 0
    if parents is not None:
        tree = 2 if isinstance(parents, torch.Tensor) and parents.dim() == 2 else 1
        _check_tensor("parents", parents, (c.layout.B, N) if tree == 2 else (N,), _I32, c.device)
    if slopes is not None:
        _check_tensor("slopes", slopes, (H,), _F32, c.device)
    return _lib.CachedAttnOptions(H, N, _left(window), tree, float(softcap), _ptr(slopes))


def _bytes(layout: _Layout, H: int, N: int, left: int) -> int:
    key = (H, N, left)
    known = layout.bytes.get(key)
    if known is None:
        n = ctypes.c_size_t(0)
        _lib.check(_lib.lib().fc_cached_attn_workspace_bytes(
            layout.ref, ctypes.byref(_lib.CachedAttnOptions(H, N, left, 0, 0.0, None)), ctypes.byref(n)))
        if len(layout.bytes) >= 256:  # (windows and batches without end)
            layout.bytes.clear()
        known = layout.bytes[key] = n.value
    return known


def cached_attention_workspace_bytes(Q: torch.Tensor, cache: KVCache, window=(-1, 0)) -> int:
    """Bytes of the caller-owned workspace ``cached_attention_(…, workspace=)`` accepts (the
    library's requirement plus 256 bytes of alignment slack; 0 when the problem needs none)."""
    if not isinstance(Q, torch.Tensor) or Q.dim() != 4:
        raise ValueError("Q must have shape (B, N, H, D)")
    c = _buffers(cache, Q.shape[0])
    n = _bytes(c.layout, Q.shape[2], Q.shape[1], _left(window))
    return n + 256 if n > 0 else 0


def cached_attention_(O: torch.Tensor, Q: torch.Tensor, cache: KVCache, lengths: torch.Tensor,
                      window: Tuple[int, int] = (-1, 0), *, counts: Optional[torch.Tensor] = None,
                      parents: Optional[torch.Tensor] = None, softcap: float = 0.0,
                      slopes: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> None:
    """``cached_attention`` into the caller's O (bfloat16, as Q)."""
    if not isinstance(Q, torch.Tensor) or Q.dim() != 4:
        raise ValueError("Q must have shape (B, N, H, D)")
    B, N, H, D = Q.shape
    c = _buffers(cache, B)
    layout, device = c.layout, c.device
    if not (D == layout.D and Q.dtype is torch.bfloat16 and Q.device == device and Q.is_contiguous() and isinstance(O, torch.Tensor)
            and O.shape == Q.shape and O.dtype is torch.bfloat16 and O.device == device and O.is_contiguous()):
        shape = (B, N, H, layout.D)
        _check_tensor("Q", Q, shape, _BF16, device)
        _check_tensor("O", O, shape, _BF16, device)
    _check_counts(c, lengths, counts, required=True)
    at = O.data_ptr()
    if at % 16:
        raise ValueError("O must start on a 16-byte boundary")
    o = _options(c, N, H, window, parents, softcap, slopes)
    nbytes = _bytes(layout, H, N, o.left)
    ws = None
    if nbytes > 0:
        if workspace is None:  # freed to this stream's pool on return, so later work on the stream comes after the kernels
            workspace = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
        else:
            _check_workspace(workspace, nbytes + 256, device)
        ws = (workspace.data_ptr() + 255) & ~255
    Q = _aligned(Q)
    _call(device, _lib.lib().fc_cached_attn, layout.ref, ctypes.byref(c.pointers), ctypes.byref(o), Q.data_ptr(), at,
          lengths.data_ptr(), _ptr(counts), _ptr(parents), ws, nbytes)


def cached_attention(Q: torch.Tensor, cache: KVCache, lengths: torch.Tensor, window: Tuple[int, int] = (-1, 0), *,
                     counts: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None, softcap: float = 0.0,
                     slopes: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest tokens over one layer's cache: Q (B, N, H, D), N from 1 to 64, for
    the tokens that ``cache_write_`` has put behind ``lengths``; bfloat16, or float32 or float16
    that is rounded to it, and the result in the same type.

    Each token sees the cache's and the new ones before it, or with ``parents`` (int32, (N,) or
    (B, N)) the cache's and its ancestors: a drafted node's parent is a node before it, -1 where
    it follows the sequence itself.  ``window`` (left, 0), ``softcap`` and ``slopes`` are those of
    ``attention``, over positions in the text (a node's is ``lengths[b]`` plus its ancestors).
    Nodes from ``counts[b]`` on get zeros; one beyond the cache's capacity, or whose
    parents are no tree's, gets NaN.  A value that is not finite is the result in its column
    for the nodes that see it, and reaches no other."""
    if isinstance(Q, torch.Tensor) and Q.dtype in (torch.float32, torch.float16):
        x = Q.to(torch.bfloat16)
        O = torch.empty_like(x)
        cached_attention_(O, x, cache, lengths, window, counts=counts, parents=parents, softcap=softcap, slopes=slopes,
                          workspace=workspace)
        return O.to(Q.dtype)
    O = torch.empty_like(Q)
    cached_attention_(O, Q, cache, lengths, window, counts=counts, parents=parents, softcap=softcap, slopes=slopes, workspace=workspace)
    return O
