"""Paged key/value cache: append with norm and rotation, and attention of new tokens over it.

The reference keeps one fixed-capacity cache row per sequence
(src/minifield_training/models/lfm2_5/decode.py:96-117); here the tokens of a
sequence lie in pages of a shared pool, listed in order by its row of
``page_table``. A call's new tokens -- one per sequence in a decode step, a
chunk of a prompt, or any mixture -- are concatenated, sequence b's being
rows ``cu_q[b]`` to ``cu_q[b + 1]`` (rows behind the last are padding and left
as they were), and are the last of its ``seq_lens[b]`` tokens.
"""

import ctypes
import functools

from .. import _lib
from ..device import DeviceArray, as_device, stream_workspace
from .rotary import DTYPE_CODES, check_out, projection


class PagedCache:
    """Key and value pools [num_pages, page_size, kv_heads, head_dim] of one layer.

    ``head_major`` pools are [num_pages, kv_heads, page_size, head_dim].
    """

    __slots__ = ("keys", "values", "head_major", "num_pages", "page_size", "kv_heads", "head_dim", "dtype")

    def __init__(self, keys: DeviceArray, values: DeviceArray, *, head_major: bool = False):
        if keys.shape != values.shape or keys.dtype != values.dtype or keys.ndim != 4:
            raise ValueError("key and value pages must be two [num_pages, page_size, kv_heads, head_dim] arrays")
        if keys.dtype not in ("bfloat16", "float16"):
            raise TypeError(f"pages must be bfloat16 or float16, got {keys.dtype}")
        self.keys, self.values, self.head_major, self.dtype = keys, values, bool(head_major), keys.dtype
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = keys.shape
        if head_major:
            self.page_size, self.kv_heads = self.kv_heads, self.page_size
        if self.page_size < 8 or self.page_size & (self.page_size - 1):
            raise ValueError("page_size must be a power of two of at least 8")

    @classmethod
    def zeros(cls, num_pages, page_size, kv_heads, head_dim, dtype="bfloat16", *, head_major=False):
        """Pools of zeros that any stream may use once this returns."""
        shape = (num_pages, kv_heads, page_size, head_dim) if head_major else (num_pages, page_size, kv_heads,
                                                                               head_dim)
        cache = cls(DeviceArray.zeros(shape, dtype), DeviceArray.zeros(shape, dtype), head_major=head_major)
        # Created streams do not wait for the default one: a first append could run before the clearing.
        _lib.call("mfb_stream_sync", None)
        return cache


def _sequences(cu_q, seq_lens, page_table, stream):
    cu_q, seq_lens = as_device(cu_q, "int32", stream), as_device(seq_lens, "int32", stream)
    page_table = as_device(page_table, "int32", stream)
    if seq_lens.ndim != 1 or cu_q.shape != (seq_lens.shape[0] + 1,):
        raise ValueError("seq_lens must be [batch] and cu_q [batch + 1]")
    if page_table.ndim != 2 or page_table.shape[0] != seq_lens.shape[0]:
        raise ValueError("page_table must be [batch, max_pages]")
    return cu_q, seq_lens, page_table


def paged_append(qkv, cache: PagedCache, cu_q, seq_lens, page_table, *, heads, freqs, interleaved=False,
                 amplitude=1.0, q_weight=None, k_weight=None, eps=1e-5, out=None, stream=None):
    """q [N, heads, D] of the projection ``qkv`` [N, (heads + 2 kv_heads) D]; k and v go to their pages.

    Norm and rotation as in ``rotary.qk_rotary_fwd``, at each token's place in
    its sequence. A token without a page (entry outside the pool, or behind
    the table) is not stored. A pool or table of no pages is refused, as
    ``paged_attention`` refuses it.
    """
    n, ld, d, freqs, wq, wk = projection(qkv, heads, cache.kv_heads, cache.head_dim, freqs, q_weight, k_weight,
                                         stream)
    if qkv.dtype != cache.dtype:
        raise TypeError(f"the projection is {qkv.dtype}, the cache {cache.dtype}")
    cu_q, seq_lens, page_table = _sequences(cu_q, seq_lens, page_table, stream)
    q = check_out(out, (n, heads, d), qkv.dtype, "out")
    b, max_pages = page_table.shape
    if n and b:
        _lib.call_packed("mfb_paged_append", 0, qkv.ptr, ld, wq.ptr if wq is not None else 0,
                  wk.ptr if wk is not None else 0, freqs.ptr, cu_q.ptr, seq_lens.ptr, page_table.ptr, q.ptr,
                  cache.keys.ptr, cache.values.ptr, n, b, max_pages, cache.num_pages, cache.page_size, heads,
                  cache.kv_heads, d, 2 * freqs.shape[0], int(interleaved), int(cache.head_major),
                  DTYPE_CODES[qkv.dtype], amplitude, eps, stream=stream)
    return q


@functools.lru_cache(maxsize=4096)
def paged_attention_workspace_size(tokens, batch, max_q, heads, kv_heads, head_dim) -> int:
    """Bytes ``paged_attention`` needs for up to ``tokens`` new tokens, at most ``max_q`` of a sequence."""
    return int(_lib.lib().mfb_paged_attn_workspace_size(tokens, batch, max_q, heads, kv_heads, head_dim))


def paged_attention(q, cache: PagedCache, cu_q, seq_lens, page_table, *, max_q, scale=None, out=None, lse=None,
                    workspace=None, stream=None):
    """o [N, heads, D] of the new tokens q [N, heads, D] over the cache.

    Causal: the i-th of a sequence's n new tokens sees its first
    ``seq_lens[b] - n + i + 1`` tokens; one that sees none gets zeros. ``max_q``
    is an upper bound of any sequence's new tokens (1 in a decode step).
    ``scale`` (positive) defaults to head_dim ** -0.5. ``lse`` (float32 [N, heads], optional) receives the
    natural log-sum-exp of the scaled scores. Calls on one ``workspace``
    (``paged_attention_workspace_size`` bytes) must not overlap; the default
    one belongs to the device and stream, and a captured call needs its own.

    A sequence's keys and values must be finite: one that is not reaches the
    queries of its chunk up to 128 keys before it (behind the sequence anything
    may lie). What contradicts itself on the device (lengths, page ids) is
    clamped and recorded for ``paged_attention_status``.
    """
    q = as_device(q, cache.dtype, stream)
    if q.ndim != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    n, heads, d = q.shape
    if d != cache.head_dim:
        raise ValueError("Paged attention query/KV shapes are incompatible")
    if heads % cache.kv_heads:
        raise ValueError("Query heads must be divisible by KV heads")
    cu_q, seq_lens, page_table = _sequences(cu_q, seq_lens, page_table, stream)
    max_q = int(max_q)
    if max_q <= 0:
        raise ValueError("max_q must be positive")
    out = check_out(out, (n, heads, d), q.dtype, "out")
    if lse is not None:
        check_out(lse, (n, heads), "float32", "lse")
    b, max_pages = page_table.shape
    if n and b:
        shared = 0
        if workspace is None:
            need = paged_attention_workspace_size(n, b, max_q, heads, cache.kv_heads, d)
            workspace, shared = stream_workspace("paged attention", need, stream), _lib.PACKED_SHARED_WORKSPACE
        _lib.call_packed("mfb_paged_attn", shared, q.ptr, cache.keys.ptr, cache.values.ptr, cu_q.ptr, seq_lens.ptr, page_table.ptr,
                  out.ptr, lse.ptr if lse is not None else 0, n, b, max_q, max_pages, cache.num_pages,
                  cache.page_size, heads, cache.kv_heads, d, int(cache.head_major), DTYPE_CODES[q.dtype],
                  d ** -0.5 if scale is None else float(scale), workspace.ptr, workspace.nbytes, stream=stream)
    return out


def paged_attention_status() -> int:
    """Reads and clears the device status word: 0, or what a call clamped or gave up on (see mfb200.h)."""
    code = ctypes.c_int()
    _lib.call("mfb_paged_attn_status", ctypes.byref(code))
    return code.value


__all__ = ["PagedCache", "paged_append", "paged_attention", "paged_attention_status",
           "paged_attention_workspace_size"]
