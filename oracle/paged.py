"""Rotary positions with head norms, paged caches and logit controls in float64 (TEST INFRASTRUCTURE ONLY).

Plain loops over heads, sequences and rows from the operators' definitions; the
inputs are the exact (already rounded) values the kernels read. ``*_bound``
values are what an error bound scales with, returned beside the result.
"""

import numpy as np


def rotation(x, position, freqs, amplitude, interleaved, inverse=False):
    """R(p) x (or its transpose) for vectors x [..., D]; the first 2 len(freqs) values turn."""
    r = 2 * len(freqs)
    angle = float(position) * np.asarray(freqs, np.float64)
    c, s = amplitude * np.cos(angle), amplitude * np.sin(angle) * (-1.0 if inverse else 1.0)
    y = np.array(x, np.float64)
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = np.array(y[..., first]), np.array(y[..., second])
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def head_forward(x, gain, position, freqs, amplitude, interleaved, eps):
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    return rotation(x, position, freqs, amplitude, interleaved)


def head_backward(x, gain, dy, position, freqs, amplitude, interleaved, eps):
    """(dx, dgain) of head_forward for one head vector."""
    du = rotation(dy, position, freqs, amplitude, interleaved, inverse=True)
    if gain is None:
        return du, None
    x = np.asarray(x, np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, w = x * r, du * gain
    return r * (w - n * (w * n).mean(-1, keepdims=True)), du * n


def split_heads(qkv, heads, kv_heads, d):
    """q, k, v heads [M, *, d] of a projection whose rows may be longer than its heads."""
    x = np.asarray(qkv, np.float64)[:, : (heads + 2 * kv_heads) * d].reshape(len(qkv), heads + 2 * kv_heads, d)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]


def cache_rows(pages, table_row, length, head_major):
    """[length, Hk, D] float64 rows of one sequence."""
    p = np.swapaxes(pages, 1, 2) if head_major else pages
    size = p.shape[1]
    return np.stack([p[table_row[j // size], j % size] for j in range(length)]).astype(np.float64) if length else \
        np.zeros((0,) + p.shape[2:])


def attention(q, keys, values, cu_q, seq_lens, table, scale, head_major=False):
    """(o, lse, spread, score): spread = sum_j p_j |v_j|, score = max_j scale sum_d |q_d k_jd| per output."""
    n, h, d = q.shape
    q = np.asarray(q, np.float64)
    o, lse = np.zeros((n, h, d)), np.full((n, h), -np.inf)
    spread, score = np.zeros((n, h, d)), np.zeros((n, h))
    for b, length in enumerate(seq_lens):
        count = cu_q[b + 1] - cu_q[b]
        k = cache_rows(keys, table[b], length, head_major) if count else None
        v = cache_rows(values, table[b], length, head_major) if count else None
        for i in range(count):
            seen = min(length - count + i + 1, length)
            if seen <= 0:
                continue
            row = cu_q[b] + i
            for head in range(h):
                kk, vv = k[:seen, head * k.shape[1] // h], v[:seen, head * k.shape[1] // h]
                s = scale * (kk @ q[row, head])
                top = s.max()
                p = np.exp(s - top)
                lse[row, head] = top + np.log(p.sum())
                p /= p.sum()
                o[row, head], spread[row, head] = p @ vv, p @ np.abs(vv)
                score[row, head] = scale * np.max(np.abs(kk) @ np.abs(q[row, head]))
    return o, lse, spread, score


def controlled_logits(logits, history=None, prompt_len=None, history_len=None, repetition=None, frequency=None,
                      presence=None, bias_ids=None, bias_values=None, mask=None, mask_rows=None):
    x = np.array(logits, np.float64)
    rows, vocab = x.shape
    for b in range(rows):
        if history is not None:
            used = history.shape[1] if history_len is None else int(np.clip(history_len[b], 0, history.shape[1]))
            prompt = 0 if prompt_len is None else int(np.clip(prompt_len[b], 0, used))
            ids = [int(t) for t in history[b, :used]]
            for t in {t for t in ids if 0 <= t < vocab}:
                if repetition is not None:
                    x[b, t] = x[b, t] / repetition[b] if x[b, t] > 0 else x[b, t] * repetition[b]
                made = ids[prompt:].count(t)
                if made:
                    x[b, t] -= (frequency[b] * made if frequency is not None else 0.0)
                    x[b, t] -= presence[b] if presence is not None else 0.0
        if bias_ids is not None:
            for t, value in {int(t): float(v) for t, v in zip(bias_ids[b], bias_values[b])}.items():
                if 0 <= t < vocab:
                    x[b, t] += value
        if mask is not None:
            m = b if mask_rows is None else int(mask_rows[b])
            if 0 <= m < len(mask):
                bits = np.unpackbits(np.ascontiguousarray(mask[m]).view(np.uint8), bitorder="little")[:vocab]
                x[b, bits == 0] = -np.inf
    return x
