"""Controls on a step's logits before sampling: penalties for repeated tokens, biases, grammar masks.

The reference hands raw FP32 logits to its caller
(src/minifield_training/models/lfm2_5/decode.py:419-466). ``process_logits``
applies the requests' controls in the pass that widens the logits to FP32.
"""

from .. import _lib
from ..device import DeviceArray, as_device
from .rotary import DTYPE_CODES, check_out


def _per_row(x, rows, dtype, what, stream):
    if x is not None:
        x = as_device(x, dtype, stream)
        if x.shape != (rows,):
            raise ValueError(f"{what} must be [rows]")
    return x


def _ptr(x):
    return x.ptr if x is not None else 0


def prepare_controls(rows, vocab, *, history=None, prompt_len=None, history_len=None, repetition=None, frequency=None,
                     presence=None, bias_ids=None, bias_values=None, mask=None, mask_rows=None, stream=None):
    """The checked controls of ``process_logits`` for [rows, vocab] logits, on the device.

    A caller that must know before its own work that they will be taken checks
    them here, then passes the result on as ``controls``.
    """
    capacity = biases = masks = 0
    if history is not None:
        history = as_device(history, "int32", stream)
        if history.ndim != 2 or history.shape[0] != rows:
            raise ValueError("history must be [rows, tokens]")
        capacity = history.shape[1]
        if capacity >= 1 << 20:
            raise ValueError(f"history of {capacity} tokens unsupported (0 to {(1 << 20) - 1})")
    elif any(x is not None for x in (prompt_len, history_len, repetition, frequency, presence)):
        raise ValueError("penalties and lengths need a history")
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values must both be given or both be None")
    if bias_ids is not None:
        bias_ids, bias_values = as_device(bias_ids, "int32", stream), as_device(bias_values, "float32", stream)
        if bias_ids.ndim != 2 or bias_ids.shape[0] != rows or bias_values.shape != bias_ids.shape:
            raise ValueError("bias_ids and bias_values must be [rows, entries]")
        biases = bias_ids.shape[1]
        if biases > 2047:
            raise ValueError(f"{biases} bias entries unsupported (0 to 2047)")
    if mask is not None:
        mask = as_device(mask, "int32", stream)
        if mask.ndim != 2 or mask.shape[1] != (vocab + 31) // 32:
            raise ValueError("mask must be [grammars, ceil(vocab / 32)]")
        masks = mask.shape[0]
        if mask_rows is None and masks < rows:
            raise ValueError("a mask without mask_rows needs one row per logits row")
    elif mask_rows is not None:
        raise ValueError("mask_rows needs a mask")
    return (rows, vocab, history, capacity, _per_row(prompt_len, rows, "int32", "prompt_len", stream),
            _per_row(history_len, rows, "int32", "history_len", stream),
            _per_row(repetition, rows, "float32", "repetition", stream),
            _per_row(frequency, rows, "float32", "frequency", stream),
            _per_row(presence, rows, "float32", "presence", stream), bias_ids, bias_values, biases, mask,
            _per_row(mask_rows, rows, "int32", "mask_rows", stream), masks)


def process_logits(logits, *, out=None, stream=None, controls=None, **kwargs):
    """float32 [rows, vocab] logits under the rows' controls, each optional.

    ``history`` (int32 [rows, n]) holds each row's token ids: the first
    ``prompt_len`` of the prompt, then the generated ones, ``history_len`` in
    all (defaults 0 and n; ids outside the vocabulary count for nothing). In
    this order, for a token t of a row:

    - ``repetition`` r (float32 [rows]): x / r if x > 0 else x * r, where t is in the history;
    - ``frequency`` f, ``presence`` p: x - f * (times generated) - p * (generated at all);
    - ``bias_ids``, ``bias_values`` (int32, float32 [rows, k]): x + the value at
      t's id; of equal ids the last counts, ids outside the vocabulary pad;
    - ``mask`` (int32 [grammars, ceil(vocab / 32)], bit t % 32 of word t // 32):
      x = -inf where the bit is 0. ``mask_rows`` (int32 [rows]) picks each
      row's grammar (default: row i's is i); an index outside leaves it free.

    ``logits`` are bfloat16, float16 or float32; float32 logits may be ``out``.
    ``controls`` are ``prepare_controls``' in place of these arguments.
    """
    if not isinstance(logits, DeviceArray):
        logits = as_device(logits, "float32", stream)
    if logits.ndim != 2 or logits.dtype not in DTYPE_CODES:
        raise ValueError("logits must be [rows, vocab] in bfloat16, float16 or float32")
    rows, vocab = logits.shape
    out = check_out(out, (rows, vocab), "float32", "out")
    if controls is None:
        controls = prepare_controls(rows, vocab, stream=stream, **kwargs)
    elif kwargs:
        raise TypeError("prepared controls take no further arguments")
    (r, v, history, capacity, prompt_len, history_len, repetition, frequency, presence, bias_ids, bias_values, biases,
     mask, mask_rows, masks) = controls
    if r != rows or v != vocab:
        raise ValueError(f"controls were prepared for [{r}, {v}] logits")
    if rows and vocab:
        _lib.call_packed("mfb_logits_process", 0, logits.ptr, DTYPE_CODES[logits.dtype], _ptr(history), capacity,
                         _ptr(prompt_len), _ptr(history_len), _ptr(repetition), _ptr(frequency), _ptr(presence),
                         _ptr(bias_ids), _ptr(bias_values), biases, _ptr(mask), _ptr(mask_rows), masks, out.ptr, rows,
                         vocab, stream=stream)
    return out


__all__ = ["prepare_controls", "process_logits"]
