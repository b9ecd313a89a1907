"""Rotary positions and head norms of a fused q|k|v projection, forward and backward.

The general form of the reference's ``apply_rotary``
(src/minifield_training/kernels/rotary.py:7-39) after the per-head q/k RMSNorm
of ``project_qkv`` (layers/attention.py:61-77): heads of 64 or 128, bf16 or
fp16, half or interleaved pairs, a rotated part of the head, frequencies scaled
for long contexts, with or without gains. The arithmetic is FP32 and rounded
once at the output; the reference's own 64-wide bf16 graph, rounded step by
step, is ``mfb_qknorm_rope_fwd`` / ``_bwd`` (models.encoder).
"""

import functools
import math

import numpy as np

from .. import _lib
from ..device import DeviceArray, as_device, stream_workspace

DTYPE_CODES = {"bfloat16": _lib.DTYPE_BF16, "float16": _lib.DTYPE_F16, "float32": _lib.DTYPE_F32}


def rotary_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None):
    """``(freqs, amplitude)``: float32 [rotary_dim / 2] radians per position, and the factor on cos and sin.

    Unscaled: theta ** (-2i / rotary_dim) (kernels/rotary.py:31-33), amplitude
    1. ``scaling`` stretches the positions a model was trained on by ``factor``:

    - ``{"kind": "linear", "factor": f}``: every frequency divided by f;
    - ``{"kind": "ntk", "factor": f}``: theta * f ** (R / (R - 2)), which keeps
      the fastest pair and divides the slowest frequency by f;
    - ``{"kind": "yarn", "factor": f, "original_length": n}`` (``beta_fast`` 32,
      ``beta_slow`` 1): pairs that turn at least beta_fast times over n
      positions are kept, those that turn at most beta_slow times are divided
      by f, with a linear ramp over the pair index between; amplitude
      1 + 0.1 ln f.
    """
    r = int(rotary_dim)
    if r <= 0 or r % 2:
        raise ValueError("rotary_dim must be a positive even number")
    theta = float(theta)
    if not theta > 1.0:
        raise ValueError("theta must be above 1")
    index = np.arange(r // 2, dtype=np.float64)
    if scaling is None:
        return (theta ** (-2.0 * index / r)).astype(np.float32), 1.0
    kind, factor = scaling.get("kind"), float(scaling.get("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError("the scaling factor must be at least 1")
    base = theta ** (-2.0 * index / r)
    if kind == "linear":
        return (base / factor).astype(np.float32), 1.0
    if kind == "ntk":
        if r == 2:
            raise ValueError("ntk scaling needs a rotary_dim above 2")
        return ((theta * factor ** (r / (r - 2.0))) ** (-2.0 * index / r)).astype(np.float32), 1.0
    if kind == "yarn":
        length = float(scaling["original_length"])

        def pair_turning(turns):  # the (fractional) pair that turns this often over the original length
            return r * math.log(length / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low = max(math.floor(pair_turning(scaling.get("beta_fast", 32.0))), 0)
        # May lie behind the last pair, which then turns more than beta_slow times.
        high = min(math.ceil(pair_turning(scaling.get("beta_slow", 1.0))), r - 1)
        ramp = np.clip((index - low) / max(high - low, 1e-3), 0.0, 1.0)
        return (base * (1.0 - ramp) + base / factor * ramp).astype(np.float32), 1.0 + 0.1 * math.log(factor)
    raise ValueError(f"Unsupported rotary scaling: {kind}")


def projection(qkv, heads, kv_heads, head_dim, freqs, q_weight, k_weight, stream):
    """Checked (qkv, rows, row stride, head_dim, freqs, gains) of a fused projection [..., (H + 2 Hk) D]."""
    if not isinstance(qkv, DeviceArray):
        raise TypeError("qkv must be a device array (bfloat16 or float16)")
    if qkv.dtype not in ("bfloat16", "float16"):
        raise TypeError(f"expected a bfloat16 or float16 projection, got {qkv.dtype}")
    if qkv.ndim < 2 or heads <= 0 or kv_heads <= 0:
        raise ValueError("qkv must be [tokens, (heads + 2 kv_heads) head_dim]")
    ld = qkv.shape[-1]
    if head_dim is None:
        if ld % (heads + 2 * kv_heads):
            raise ValueError("qkv columns are not (heads + 2 kv_heads) whole heads; pass head_dim")
        head_dim = ld // (heads + 2 * kv_heads)
    rows = 1
    for n in qkv.shape[:-1]:
        rows *= n
    freqs = as_device(freqs, "float32", stream)
    if freqs.ndim != 1 or 2 * freqs.shape[0] > head_dim:
        raise ValueError("freqs must be [rotary_dim / 2] with rotary_dim up to head_dim")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight must both be given or both be None")
    if q_weight is not None:
        q_weight, k_weight = as_device(q_weight, "float32", stream), as_device(k_weight, "float32", stream)
        if q_weight.shape != (head_dim,) or k_weight.shape != (head_dim,):
            raise ValueError("q_weight and k_weight must be [head_dim]")
    return rows, ld, head_dim, freqs, q_weight, k_weight


def check_out(x, shape, dtype, what):
    """``x`` as an output of ``shape``; a new array where it is None."""
    if x is None:
        return DeviceArray(shape, dtype)
    if x.dtype != dtype or x.shape != shape:
        raise ValueError(f"{what} must be a {dtype} device array of shape {shape}")
    return x


def _ptr(x):
    return x.ptr if x is not None else 0


def qk_rotary_fwd(qkv, positions, freqs, *, heads, kv_heads, head_dim=None, interleaved=False, amplitude=1.0,
                  q_weight=None, k_weight=None, eps=1e-5, out=None, stream=None):
    """``(q, k, v)`` [M, heads, D], [M, kv_heads, D] x 2 of the projection ``qkv`` [..., (heads + 2 kv_heads) D].

    With gains, q and k heads are RMS-normalised first; then their first
    ``2 len(freqs)`` values are rotated by ``positions`` (int32, one per token).
    ``out`` takes the three outputs; its third may be None to leave v uncopied.
    """
    m, ld, d, freqs, wq, wk = projection(qkv, heads, kv_heads, head_dim, freqs, q_weight, k_weight, stream)
    positions = as_device(positions, "int32", stream)
    if positions.size != m:
        raise ValueError("positions must hold one position per token")
    q, k, v = out if out is not None else (None, None, None)
    q = check_out(q, (m, heads, d), qkv.dtype, "q")
    k = check_out(k, (m, kv_heads, d), qkv.dtype, "k")
    v = check_out(v, (m, kv_heads, d), qkv.dtype, "v") if out is None or v is not None else None
    if m:
        _lib.call_packed("mfb_qk_rotary_fwd", 0, qkv.ptr, ld, _ptr(wq), _ptr(wk), positions.ptr, freqs.ptr, q.ptr, k.ptr,
                  _ptr(v), m, heads, kv_heads, d, 2 * freqs.shape[0], int(interleaved), DTYPE_CODES[qkv.dtype],
                  amplitude, eps, stream=stream)
    return q, k, v


@functools.lru_cache(maxsize=None)
def _workspace_size(head_dim):
    return _lib.lib().mfb_qk_rotary_workspace_size(head_dim)


def qk_rotary_bwd(qkv, positions, freqs, dq, dk, dv, *, head_dim=None, interleaved=False, amplitude=1.0,
                  q_weight=None, k_weight=None, eps=1e-5, out=None, weight_grads=None, accumulate=False,
                  workspace=None, stream=None):
    """``(dqkv, dq_weight, dk_weight)`` of ``qk_rotary_fwd`` for upstream dq [M, H, D], dk and dv [M, Hk, D].

    The gain gradients (float32 [D]) are new arrays, or ``weight_grads`` =
    (dq_weight, dk_weight), written or (``accumulate``) added to; None without
    gains. ``out`` may be ``qkv`` itself. Columns behind the heads have no
    gradient: zeros in a new dqkv, left as they were in ``out``. A captured call needs its own
    ``workspace`` (``mfb_qk_rotary_workspace_size(head_dim)`` bytes).
    """
    for x in (dq, dk, dv):
        if not isinstance(x, DeviceArray) or x.dtype != qkv.dtype or x.ndim < 2:
            raise ValueError("dq, dk and dv must be device arrays of the projection's dtype")
    heads, kv_heads = dq.shape[-2], dk.shape[-2]
    m, ld, d, freqs, wq, wk = projection(qkv, heads, kv_heads, head_dim, freqs, q_weight, k_weight, stream)
    positions = as_device(positions, "int32", stream)
    if positions.size != m:
        raise ValueError("positions must hold one position per token")
    if dq.size != m * heads * d or dk.size != m * kv_heads * d or dk.shape != dv.shape:
        raise ValueError("dq, dk and dv must match the projection's heads")
    if wq is None and (weight_grads is not None or accumulate):
        raise ValueError("gain gradients need the gains")
    if accumulate and (weight_grads is None or any(g is None for g in weight_grads)):
        raise ValueError("accumulate needs weight_grads to add to")
    dqkv = check_out(out, qkv.shape, qkv.dtype, "out")
    if out is None and ld > (heads + 2 * kv_heads) * d:
        _lib.call("mfb_memset", dqkv.ptr, 0, dqkv.nbytes, stream)
    dwq = dwk = ws = None
    shared = 0
    if wq is not None:
        dwq, dwk = weight_grads if weight_grads is not None else (None, None)
        dwq, dwk = check_out(dwq, (d,), "float32", "dq_weight"), check_out(dwk, (d,), "float32", "dk_weight")
        if workspace is None:
            ws, shared = stream_workspace("rotary", _workspace_size(d), stream), _lib.PACKED_SHARED_WORKSPACE
        else:
            ws = workspace
    if m:
        _lib.call_packed("mfb_qk_rotary_bwd", shared, qkv.ptr, ld, _ptr(wq), _ptr(wk), positions.ptr, freqs.ptr, dq.ptr, dk.ptr,
                  dv.ptr, dqkv.ptr, _ptr(dwq), _ptr(dwk), int(accumulate), m, heads, kv_heads, d,
                  2 * freqs.shape[0], int(interleaved), DTYPE_CODES[qkv.dtype], amplitude, eps, _ptr(ws),
                  ws.nbytes if ws is not None else 0, stream=stream)
    elif dwq is not None and not accumulate:
        for x in (dwq, dwk):
            _lib.call("mfb_memset", x.ptr, 0, x.nbytes, stream)
    return dqkv, dwq, dwk


__all__ = ["qk_rotary_bwd", "qk_rotary_fwd", "rotary_frequencies"]
