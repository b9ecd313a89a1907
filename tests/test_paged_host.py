"""Host side of the rotary, paged-cache and logit operators (no GPU): frequencies, refusals, the oracle itself.

Every refusal happens before any device work: the arrays here hold addresses
that nothing may touch.
"""

import ctypes
import math

import numpy as np
import pytest

from minifield_training_b200 import _lib
from minifield_training_b200.device import DeviceArray
from minifield_training_b200.kernels import logits as lg
from minifield_training_b200.kernels import paged, rotary
from oracle import paged as op


def fake(shape, dtype, ptr=1 << 20):
    return DeviceArray(shape, dtype, ptr=ptr, owner=False)


def test_frequencies_follow_their_definitions():
    f, a = rotary.rotary_frequencies(64, 1e6)
    np.testing.assert_allclose(f, 1e6 ** (-np.arange(0, 64, 2) / 64), rtol=2 ** -23)
    assert f.dtype == np.float32 and a == 1.0
    lin, a = rotary.rotary_frequencies(64, 1e4, {"kind": "linear", "factor": 4})
    np.testing.assert_allclose(lin, rotary.rotary_frequencies(64, 1e4)[0] / 4, rtol=2 ** -22)
    ntk, _ = rotary.rotary_frequencies(64, 1e4, {"kind": "ntk", "factor": 8})
    base = rotary.rotary_frequencies(64, 1e4)[0]
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(base[-1] / 8, rel=1e-6)  # the ends the method fixes
    yarn, amp = rotary.rotary_frequencies(128, 1e4, {"kind": "yarn", "factor": 16, "original_length": 4096})
    base = rotary.rotary_frequencies(128, 1e4)[0]
    turns = 4096 * base / (2 * math.pi)
    assert np.array_equal(yarn[turns > 40], base[turns > 40])
    np.testing.assert_allclose(yarn[turns < 0.8], base[turns < 0.8] / 16, rtol=2 ** -22)
    assert np.all(np.diff(yarn) < 0) and amp == pytest.approx(1 + 0.1 * math.log(16))


@pytest.mark.parametrize("args", [(0, 1e4, None), (7, 1e4, None), (64, 0.5, None),
                                  (64, 1e4, {"kind": "cubic", "factor": 2}),
                                  (64, 1e4, {"kind": "linear", "factor": 0.5}),
                                  (2, 1e4, {"kind": "ntk", "factor": 2})])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(*args)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("gained", [False, True])
def test_oracle_gradient_matches_differences(interleaved, gained):
    rng = np.random.default_rng(3)
    x, dy = rng.standard_normal(64), rng.standard_normal(64)
    gain = 1 + 0.3 * rng.standard_normal(64) if gained else None
    freqs = rotary.rotary_frequencies(32, 1e4)[0]
    args = (17, freqs, 1.1, interleaved, 1e-5)
    dx, dgain = op.head_backward(x, gain, dy, *args)
    loss = lambda x, g: float(dy @ op.head_forward(x, g, *args))  # noqa: E731
    for i in range(0, 64, 5):
        e = np.zeros(64)
        e[i] = 1e-5
        assert dx[i] == pytest.approx((loss(x + e, gain) - loss(x - e, gain)) / 2e-5, abs=1e-7)
        if gained:
            assert dgain[i] == pytest.approx((loss(x, gain + e) - loss(x, gain - e)) / 2e-5, abs=1e-7)


def rotary_call(**kw):
    a = dict(qkv=fake((4, 32 * 64), "bfloat16"), positions=fake((4,), "int32"), freqs=fake((32,), "float32"),
             heads=16, kv_heads=8, out=(fake((4, 16, 64), "bfloat16"), fake((4, 8, 64), "bfloat16"), None))
    a.update(kw)
    return rotary.qk_rotary_fwd(a.pop("qkv"), a.pop("positions"), a.pop("freqs"), **a)


@pytest.mark.parametrize("kw, match", [
    (dict(qkv=fake((4, 2048), "float32")), "bfloat16 or float16"),
    (dict(qkv=fake((4, 2050), "bfloat16")), "whole heads"),
    (dict(qkv=fake((4, 32 * 96), "bfloat16"), out=(fake((4, 16, 96), "bfloat16"), fake((4, 8, 96), "bfloat16"), None)),
     "head_dim 96"),
    (dict(positions=fake((5,), "int32")), "one position per token"),
    (dict(freqs=fake((33,), "float32")), "up to head_dim"),
    (dict(freqs=fake((12,), "float32")), "multiple of 16"),
    (dict(q_weight=fake((64,), "float32")), "both be given"),
    (dict(q_weight=fake((32,), "float32"), k_weight=fake((32,), "float32")), "head_dim"),
    (dict(out=(fake((4, 16, 64), "float16"), None, None)), "q must be"),
    (dict(qkv=fake((4, 2048), "bfloat16", ptr=(1 << 20) + 8)), "16-byte aligned"),
])
def test_rotary_refuses(kw, match):
    with pytest.raises((ValueError, TypeError), match=match):
        rotary_call(**kw)


def test_rotary_backward_refuses():
    qkv, pos, f = fake((4, 2048), "bfloat16"), fake((4,), "int32"), fake((32,), "float32")
    dq, dk = fake((4, 16, 64), "bfloat16"), fake((4, 8, 64), "bfloat16")
    w, out = fake((64,), "float32"), fake((4, 2048), "bfloat16")
    with pytest.raises(ValueError, match="match the projection"):
        rotary.qk_rotary_bwd(qkv, pos, f, fake((3, 16, 64), "bfloat16"), dk, dk, out=out)
    with pytest.raises(ValueError, match="dtype"):
        rotary.qk_rotary_bwd(qkv, pos, f, dq, dk, fake((4, 8, 64), "float16"), out=out)
    with pytest.raises(ValueError, match="need the gains"):
        rotary.qk_rotary_bwd(qkv, pos, f, dq, dk, dk, out=out, weight_grads=(w, w))
    with pytest.raises(ValueError, match="to add to"):
        rotary.qk_rotary_bwd(qkv, pos, f, dq, dk, dk, out=out, q_weight=w, k_weight=w, accumulate=True)
    with pytest.raises(RuntimeError, match="workspace needs"):
        rotary.qk_rotary_bwd(qkv, pos, f, dq, dk, dk, out=out, q_weight=w, k_weight=w, weight_grads=(w, w),
                             workspace=fake((16,), "uint8"))


def append_call(**kw):
    cache = kw.pop("cache", None) or paged.PagedCache(*[fake((9, 16, 8, 64), "bfloat16")] * 2)
    a = dict(qkv=fake((4, 2048), "bfloat16"), cu_q=fake((3,), "int32"), seq_lens=fake((2,), "int32"),
             table=fake((2, 5), "int32"), heads=16, freqs=fake((32,), "float32"), out=fake((4, 16, 64), "bfloat16"))
    a.update(kw)
    return paged.paged_append(a.pop("qkv"), cache, a.pop("cu_q"), a.pop("seq_lens"), a.pop("table"), **a)


@pytest.mark.parametrize("kw, match", [
    (dict(qkv=fake((4, 2048), "float16"), out=fake((4, 16, 64), "float16")), "the cache bfloat16"),
    (dict(cu_q=fake((2,), "int32")), r"cu_q \[batch \+ 1\]"),
    (dict(table=fake((3, 5), "int32")), "page_table"),
    (dict(out=fake((4, 16, 32), "bfloat16")), "out must be"),
    (dict(seq_lens=fake((2,), "float32")), "expected int32"),
])
def test_append_refuses(kw, match):
    with pytest.raises((ValueError, TypeError), match=match):
        append_call(**kw)


def attention_call(**kw):
    cache = kw.pop("cache", None) or paged.PagedCache(*[fake((9, 16, 8, 64), "bfloat16")] * 2)
    a = dict(q=fake((4, 16, 64), "bfloat16"), cu_q=fake((3,), "int32"), seq_lens=fake((2,), "int32"),
             table=fake((2, 5), "int32"), max_q=2, out=fake((4, 16, 64), "bfloat16"), workspace=fake((16,), "uint8"))
    a.update(kw)
    return paged.paged_attention(a.pop("q"), cache, a.pop("cu_q"), a.pop("seq_lens"), a.pop("table"), **a)


@pytest.mark.parametrize("kw, match", [
    (dict(), "workspace needs"),
    (dict(q=fake((4, 12, 64), "bfloat16")), "divisible"),
    (dict(q=fake((4, 16, 128), "bfloat16")), "incompatible"),
    (dict(q=fake((4, 16, 64), "float16")), "expected bfloat16"),
    (dict(max_q=0), "max_q"),
    (dict(lse=fake((4, 8), "float32")), "lse must be"),
    (dict(q=fake((4, 16, 64), "bfloat16", ptr=(1 << 20) + 2)), "16-byte aligned"),
    (dict(table=fake((2, 1 << 28), "int32")), "positions"),
    (dict(scale=0.0), "positive and finite"),
    (dict(scale=-0.125), "positive and finite"),
    (dict(scale=float("nan")), "positive and finite"),
    (dict(cu_q=fake((8001,), "int32"), seq_lens=fake((8000,), "int32"), table=fake((8000, 1 << 20), "int32")),
     "exceeds 2"),
    (dict(table=fake((2, 1 << 26), "int32"), q=fake((1 << 20, 16, 64), "bfloat16"), max_q=1 << 19,
          out=fake((1 << 20, 16, 64), "bfloat16")), "exceeds 2"),
    (dict(cache=paged.PagedCache(*[fake((9, 16, 8, 32), "bfloat16")] * 2), q=fake((4, 16, 32), "bfloat16"),
          out=fake((4, 16, 32), "bfloat16")), "head_dim 32"),
])
def test_attention_refuses(kw, match):
    with pytest.raises((ValueError, TypeError, RuntimeError), match=match):
        attention_call(**kw)


def test_cache_refuses():
    with pytest.raises(ValueError, match="power of two"):
        paged.PagedCache(*[fake((9, 12, 8, 64), "bfloat16")] * 2)
    with pytest.raises(ValueError, match="power of two"):
        paged.PagedCache(*[fake((9, 8, 4, 64), "bfloat16")] * 2, head_major=True)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        paged.PagedCache(*[fake((9, 16, 8, 64), "float32")] * 2)
    with pytest.raises(ValueError, match="two"):
        paged.PagedCache(fake((9, 16, 8, 64), "bfloat16"), fake((8, 16, 8, 64), "bfloat16"))
    hm = paged.PagedCache(*[fake((9, 8, 16, 64), "bfloat16")] * 2, head_major=True)
    assert (hm.page_size, hm.kv_heads) == (16, 8)


def test_empty_calls_launch_nothing():
    """No tokens or no sequences: outputs untouched, nothing launched (there is no device here)."""
    q = append_call(qkv=fake((0, 2048), "bfloat16"), out=fake((0, 16, 64), "bfloat16"))
    assert q.shape == (0, 16, 64)
    o = attention_call(q=fake((0, 16, 64), "bfloat16"), out=fake((0, 16, 64), "bfloat16"))
    assert o.shape == (0, 16, 64)
    q, k, _ = rotary_call(qkv=fake((0, 2048), "bfloat16"), positions=fake((0,), "int32"),
                          out=(fake((0, 16, 64), "bfloat16"), fake((0, 8, 64), "bfloat16"), None))
    assert q.shape == (0, 16, 64) and k.shape == (0, 8, 64)
    out = fake((0, 100), "float32")
    assert lg.process_logits(fake((0, 100), "bfloat16"), out=out) is out


@pytest.mark.parametrize("kw, match", [
    (dict(out=fake((2, 99), "float32")), "out must be"),
    (dict(repetition=fake((2,), "float32")), "need a history"),
    (dict(history=fake((3, 8), "int32")), "history must be"),
    (dict(history=fake((2, 1 << 20), "int32")), "history of"),
    (dict(history=fake((2, 8), "int32"), presence=fake((3,), "float32")), "presence must be"),
    (dict(bias_ids=fake((2, 3), "int32")), "both be given"),
    (dict(bias_ids=fake((2, 2048), "int32"), bias_values=fake((2, 2048), "float32")), "bias entries"),
    (dict(mask=fake((2, 3), "int32")), "mask must be"),
    (dict(mask=fake((1, 4), "int32")), "one row per logits row"),
    (dict(mask_rows=fake((2,), "int32")), "needs a mask"),
    (dict(logits=fake((2, 100), "int32")), "logits must be"),
    (dict(logits=fake((2, 100), "bfloat16", ptr=(1 << 20) + 2)), "16-byte aligned"),
    (dict(logits=fake((1, (1 << 24) + 1), "bfloat16"), out=fake((1, (1 << 24) + 1), "float32")), "vocabulary"),
])
def test_logits_refuse(kw, match):
    a = dict(logits=fake((2, 100), "bfloat16"), out=fake((2, 100), "float32"))
    a.update(kw)
    with pytest.raises((ValueError, TypeError), match=match):
        lg.process_logits(a.pop("logits"), **a)


def test_workspace_sizes_cover_odd_shapes():
    size = _lib.lib().mfb_paged_attn_workspace_size
    assert size(4, 2, 2, 16, 8, 64) > 0
    assert size(4, 2, 2, 15, 8, 64) == 0 and size(0, 2, 2, 16, 8, 64) == 0 and size(4, 2, 2, 16 * 129, 16, 64) == 0
    assert size(8192, 7, 4096, 16, 8, 64) < 1 << 26
    flag = ctypes.c_int(5)
    assert _lib.lib().mfb_stream_is_capturing(None, None) == _lib.ERR_INVALID
    assert flag.value == 5


@pytest.mark.parametrize("kw, match", [
    (dict(batch_size=0), "batch_size"),
    (dict(batch_size=8193), "8192 rows"),
    (dict(num_pages=-1), "num_pages"),
    (dict(num_pages=True), "num_pages"),
    (dict(page_size=12), "power of two"),
    (dict(page_size=4), "power of two"),
    (dict(max_pages=0), "max_pages"),
])
def test_paged_state_refuses(kw, match):
    from minifield_training_b200 import workloads
    from minifield_training_b200.models import decode
    with pytest.raises(ValueError, match=match):
        decode.new_paged_state(workloads.DECODER, **{**dict(batch_size=2, num_pages=4), **kw})


def test_prepared_controls_refuse():
    with pytest.raises(ValueError, match="history must be"):
        lg.prepare_controls(2, 100, history=fake((3, 8), "int32"))
    ready = lg.prepare_controls(2, 100, history=fake((2, 8), "int32"))
    logits, out = fake((3, 100), "bfloat16"), fake((3, 100), "float32")
    with pytest.raises(ValueError, match="prepared for"):
        lg.process_logits(logits, out=out, controls=ready)
    with pytest.raises(TypeError, match="no further"):
        lg.process_logits(fake((2, 100), "bfloat16"), out=fake((2, 100), "float32"), controls=ready,
                          mask=fake((2, 4), "int32"))


def test_packed_calls_refuse():
    """Integers past their parameter's 32 bits and a missing block are refused, not truncated."""
    for large in (1 << 31, 1 << 40, (1 << 32) + 2):
        with pytest.raises(ValueError, match="out of range"):
            attention_call(max_q=large)
    with pytest.raises(ValueError, match="out of range"):
        append_call(heads=16, table=fake((2, 1 << 33), "int32"))
    for name in ("mfb_qk_rotary_fwd", "mfb_qk_rotary_bwd", "mfb_paged_append", "mfb_paged_attn", "mfb_logits_process"):
        assert getattr(_lib.lib(), name + "_packed")(None) == _lib.ERR_INVALID
        assert name in _lib.last_error()
