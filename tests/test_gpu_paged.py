"""Rotary, paged-cache and logit operators on the GPU against oracle/paged.py in float64.

Tolerances count roundings. u = 2^-8 (bf16) or 2^-11 (fp16) is half a step of
the stored type, relative to the value. FP32 arithmetic adds a few 2^-24 of
the magnitudes that enter a sum.

- Rotary: |error| <= u |y| + 2^-19 (|a| + |b|) with a, b the rotated pair (about
  20 FP32 operations, and angles good to 2^-20 rad).
- Attention: probabilities are rounded once to the cache's type, |error| <=
  u |o| + (u + 4 e) sum_j p_j |v_j|, where e = 2^-20 max_j |scaled score terms|
  covers the FP32 score (D products; tensor-core sums may truncate) and 2^-18
  the exponential and the joins; fp16 probabilities below 2^-14 round by 2^-25
  of the largest, n keys of them.
"""

import ctypes

import ml_dtypes
import numpy as np
import pytest

from oracle import paged as op
from tests.gpu_env import require_gpu

pytestmark = pytest.mark.gpu
NP = {"bfloat16": np.dtype(ml_dtypes.bfloat16), "float16": np.dtype(np.float16), "float32": np.dtype(np.float32)}
U = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def dev(x, dtype=None):
    from minifield_training_b200.device import DeviceArray
    return DeviceArray.from_numpy(x, dtype)


def normal(rng, shape, dtype):
    return rng.standard_normal(shape, dtype=np.float32).astype(NP[dtype])


# ---- rotary ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("m, h, hk, d, part, interleaved, gains, far, dtype, pad", [
    (1, 16, 8, 64, 64, False, True, 0, "bfloat16", 0),
    (37, 16, 8, 64, 64, False, True, 0, "bfloat16", 8),
    (5, 3, 1, 64, 16, False, True, 1 << 20, "float16", 0),
    (130, 12, 4, 128, 64, True, False, 1 << 24, "float16", 0),
    (257, 5, 5, 128, 128, False, True, 3000, "bfloat16", 24),
    (33, 1, 1, 128, 96, True, True, 0, "bfloat16", 0),
    (9, 7, 2, 64, 0, False, True, 0, "float16", 0),
    (3000, 4, 2, 64, 32, False, False, (1 << 31) - 4000, "bfloat16", 0),
    (3000, 4, 2, 64, 64, True, True, -5000, "bfloat16", 0),
])
def test_rotary_forward_and_backward(m, h, hk, d, part, interleaved, gains, far, dtype, pad):
    require_gpu()
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import rotary

    rng = np.random.default_rng(m + d + part)
    ld = (h + 2 * hk) * d + pad
    qkv = normal(rng, (m, ld), dtype)
    qkv[0, :d] = 0  # a head of zeros
    dq, dk, dv = (normal(rng, (m, n, d), dtype) for n in (h, hk, hk))
    freqs = rotary.rotary_frequencies(part, 1e4)[0] if part else np.zeros(0, np.float32)
    amp = 1.25
    pos = (far + np.arange(m) % 2048).astype(np.int32)
    wq, wk = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if gains else None for _ in range(2))
    kw = dict(head_dim=d, interleaved=interleaved, amplitude=amp, q_weight=None if wq is None else dev(wq),
              k_weight=None if wk is None else dev(wk), eps=1e-5)
    a, p, f = dev(qkv, dtype), dev(pos), dev(freqs)
    q, k, v = rotary.qk_rotary_fwd(a, p, f, heads=h, kv_heads=hk, **kw)
    out = DeviceArray.from_numpy(np.full((m, ld), 7, NP[dtype]), dtype)
    base = [rng.standard_normal(d).astype(np.float32) for _ in range(2)]
    grads = tuple(dev(x) for x in base) if gains else None
    dqkv, dwq, dwk = rotary.qk_rotary_bwd(a, p, f, dev(dq, dtype), dev(dk, dtype), dev(dv, dtype), out=out,
                                          weight_grads=grads, accumulate=gains, **kw)
    hq, hkk, hv = op.split_heads(qkv.astype(np.float64), h, hk, d)
    got = {"q": q.numpy(), "k": k.numpy()}
    dgot = op.split_heads(dqkv.numpy().astype(np.float64), h, hk, d)
    np.testing.assert_array_equal(v.numpy(), hv.astype(NP[dtype]))
    np.testing.assert_array_equal(dgot[2].astype(NP[dtype]), dv)
    assert np.all(dqkv.numpy()[:, (h + 2 * hk) * d:] == 7)  # columns behind the heads
    u, rows = U[dtype], range(m) if m <= 257 else list(range(0, m, 97)) + [m - 1]
    dw = [np.zeros(d), np.zeros(d)]
    dws = [np.zeros(d), np.zeros(d)]
    for which, (x, w, dy) in enumerate(((hq, wq, dq), (hkk, wk, dk))):
        for t in rows:
            y = op.head_forward(x[t], w, pos[t], freqs, amp, interleaved, 1e-5)
            mag = np.abs(y).max(-1, keepdims=True) + 1e-30
            err = np.abs(got["qk"[which]][t].astype(np.float64) - y)
            assert np.all(err <= u * np.abs(y) + 2.0 ** -18 * mag), (which, t, err.max())
        for t in range(m):
            dx, dg = op.head_backward(x[t], w, dy[t].astype(np.float64), pos[t], freqs, amp, interleaved, 1e-5)
            if gains:
                dw[which] += dg.sum(0)
                dws[which] += np.abs(dg).sum(0)
            if t in rows:
                mag = np.abs(dx).max(-1, keepdims=True)
                err = np.abs(dgot[which][t] - dx)
                # FP32 terms of the size of dy's rotation, divided by the head's norm.
                assert np.all(err <= u * np.abs(dx) + 2.0 ** -17 * mag), (which, t, err.max())
    if gains:
        for g, b, w_, s_ in zip((dwq, dwk), base, dw, dws):
            # Sums of m x heads FP32 terms in trees and per-lane runs of up to m / 64.
            assert np.all(np.abs(g.numpy() - (b + w_)) <= 2.0 ** -18 * (s_ + np.abs(b)) + 1e-6)
    else:
        assert dwq is None and dwk is None


def test_rotary_backward_in_place_and_repeatable():
    require_gpu()
    from minifield_training_b200.kernels import rotary

    rng = np.random.default_rng(0)
    m, h, hk, d = 700, 16, 8, 64
    qkv = normal(rng, (m, (h + 2 * hk) * d), "bfloat16")
    g = [dev(normal(rng, (m, n, d), "bfloat16"), "bfloat16") for n in (h, hk, hk)]
    f, p, w = dev(rotary.rotary_frequencies(d, 1e6)[0]), dev(np.arange(m, dtype=np.int32)), dev(np.ones(d, np.float32))
    a = dev(qkv, "bfloat16")
    ref = [x.numpy() for x in rotary.qk_rotary_bwd(a, p, f, *g, q_weight=w, k_weight=w)]
    same = rotary.qk_rotary_bwd(a, p, f, *g, q_weight=w, k_weight=w, out=a)
    assert same[0] is a
    for x, y in zip(same, ref):
        np.testing.assert_array_equal(x.numpy(), y)


# ---- paged cache ----------------------------------------------------------------------------------------------


def build(rng, lens, counts, h, hk, d, page, head_major, dtype, pad=0, junk=np.nan, gap=1):
    """A pool whose every row outside the sequences is ``junk``, shuffled pages, and the call's arrays."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + 2
    order = rng.permutation(total)
    shape = (total, hk, page, d) if head_major else (total, page, hk, d)
    keys, values = np.full(shape, junk, NP[dtype]), np.full(shape, junk, NP[dtype])
    table = np.full((len(lens), max(max(need), 1) + gap), -1, np.int32)
    at = 0
    for b, (n, c) in enumerate(zip(lens, need)):
        table[b, :c] = order[at:at + c]
        at += c
        for pool in (keys, values):
            view = np.swapaxes(pool, 1, 2) if head_major else pool
            rows = normal(rng, (n, hk, d), dtype)
            for i in range(c):
                part = rows[i * page:(i + 1) * page]
                view[table[b, i], : len(part)] = part
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = normal(rng, (int(cu[-1]) + pad, h, d), dtype)
    return q, keys, values, cu, np.array(lens, np.int32), table


def run_attention(q, keys, values, cu, lens, table, head_major, dtype, max_q, scale=None, stream=None, workspace=None):
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged

    cache = paged.PagedCache(dev(keys, dtype), dev(values, dtype), head_major=head_major)
    out = DeviceArray.from_numpy(np.full(q.shape, 5, NP[dtype]), dtype)
    lse = dev(np.full(q.shape[:2], 5, np.float32))
    paged.paged_attention(dev(q, dtype), cache, dev(cu), dev(lens), dev(table), max_q=max_q, out=out, lse=lse,
                          scale=scale, workspace=workspace, stream=stream)
    return out.numpy(stream), lse.numpy(stream)


def check_attention(got, lse, q, keys, values, cu, lens, table, head_major, dtype, scale):
    o, l, spread, score = op.attention(q.astype(np.float64), np.asarray(keys), np.asarray(values), cu, lens, table,
                                       scale, head_major)
    n, u = int(cu[-1]), U[dtype]
    e = 2.0 ** -20 * score[:n, :, None] + 2.0 ** -18
    tiny = 2.0 ** -25 * max(max(lens), 1) * 4 if dtype == "float16" else 0.0  # 4: the largest |v| times a margin
    err = np.abs(got[:n].astype(np.float64) - o[:n])
    bound = u * np.abs(o[:n]) + (u + 4 * e) * spread[:n] + tiny + 1e-30
    assert np.all(np.isfinite(got[:n].astype(np.float32)))
    assert np.all(err <= bound), (err.max(), np.argwhere(err > bound)[:4])
    none = np.isneginf(l[:n])
    assert np.array_equal(np.isneginf(lse[:n]), none) and not np.any(got[:n].astype(np.float32)[none])
    live = ~none
    assert np.all(np.abs(lse[:n][live] - l[:n][live]) <= 2.0 ** -20 * (8 + score[:n][live] + np.abs(l[:n][live])))
    assert np.all(got[n:].astype(np.float32) == 5) and np.all(lse[n:] == 5)  # padding: left as it was


CASES = [
    # lens, counts, H, Hk, D, page, head_major, dtype
    ([1], [1], 16, 8, 64, 16, False, "bfloat16"),
    ([200], [1], 16, 8, 64, 16, False, "bfloat16"),
    ([17, 1, 300, 0, 128, 129, 64], [1, 1, 1, 1, 1, 0, 1], 16, 8, 64, 16, False, "bfloat16"),
    ([5000, 33, 4097], [1, 1, 1], 16, 8, 64, 64, True, "float16"),
    ([700, 20, 3], [1, 1, 1], 4, 4, 128, 8, False, "bfloat16"),
    ([700, 20, 3], [8, 3, 5], 2, 1, 64, 32, False, "float16"),
    ([513, 40, 6, 90], [3, 1, 2, 0], 15, 3, 128, 128, True, "bfloat16"),
    ([260, 9], [16, 9], 6, 6, 64, 16, False, "bfloat16"),
    ([2100, 9], [8, 2], 4, 2, 128, 256, False, "float16"),
    ([257, 127, 128, 129, 256], [17, 127, 128, 129, 1], 16, 8, 64, 16, False, "bfloat16"),
    ([1000, 5, 300], [64, 5, 300], 16, 8, 64, 32, True, "float16"),
    ([1300, 90, 1, 700], [33, 90, 1, 0], 16, 4, 128, 64, False, "bfloat16"),
    ([900, 130], [70, 130], 15, 5, 128, 8, True, "float16"),
    ([300, 40], [20, 40], 7, 1, 64, 256, False, "bfloat16"),
    ([20, 3, 40], [40, 8, 33], 4, 2, 64, 16, False, "bfloat16"),  # more new tokens than cached ones: empty rows
    ([3, 0], [5, 2], 4, 2, 64, 16, False, "float16"),
    ([500], [3], 128, 1, 64, 16, False, "bfloat16"),
    ([6000], [40], 2, 1, 128, 32, False, "bfloat16"),
    ([3333], [257], 2, 2, 64, 16, False, "bfloat16"),
]


@pytest.mark.parametrize("lens, counts, h, hk, d, page, head_major, dtype", CASES)
def test_paged_attention(lens, counts, h, hk, d, page, head_major, dtype):
    require_gpu()
    from minifield_training_b200.kernels import paged

    rng = np.random.default_rng(sum(lens) + h + d)
    a = build(rng, lens, counts, h, hk, d, page, head_major, dtype, pad=3)
    paged.paged_attention_status()
    got, lse = run_attention(*a, head_major, dtype, max(counts))
    assert paged.paged_attention_status() == 0
    check_attention(got, lse, *a, head_major, dtype, d ** -0.5)
    # A looser bound on the new tokens may pick the other kernel; the answer stays.
    got2, lse2 = run_attention(*a, head_major, dtype, max(counts) + 40)
    check_attention(got2, lse2, *a, head_major, dtype, d ** -0.5)


@pytest.mark.parametrize("counts", [[1, 2], [200, 90]])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_paged_attention_sharp_scores(counts, dtype):
    """Scores up to several hundred: the running maximum moves often and far."""
    require_gpu()
    rng = np.random.default_rng(5)
    q, keys, values, cu, lens, table = build(rng, [1500, 640], counts, 4, 2, 64, 16, False, dtype)
    q = (q.astype(np.float32) * 12).astype(NP[dtype])
    view = keys[table[0, :90]]
    keys[table[0, :90]] = (view.astype(np.float32) * np.linspace(0.2, 4, 90)[:, None, None, None]).astype(NP[dtype])
    got, lse = run_attention(q, keys, values, cu, lens, table, False, dtype, max(counts), scale=0.25)
    check_attention(got, lse, q, keys, values, cu, lens, table, False, dtype, 0.25)


@pytest.mark.parametrize("count", [1, 100])
def test_paged_attention_constant_values(count):
    """Equal values: whatever the weights, the average is that value to one rounding of P and one of o."""
    require_gpu()
    rng = np.random.default_rng(6)
    q, keys, values, cu, lens, table = build(rng, [3000], [count], 16, 8, 64, 16, False, "bfloat16")
    values[:] = np.float32(1.5)
    got, _ = run_attention(q, keys, values, cu, lens, table, False, "bfloat16", count)
    assert np.all(np.abs(got.astype(np.float32) - 1.5) <= 1.5 * 2 * 2.0 ** -8)


@pytest.mark.parametrize("count", [1, 60])
def test_paged_attention_beyond_2_31_elements(count):
    """Pages past 2^31 elements (and 2^32 bytes) of the pool."""
    require_gpu()
    from minifield_training_b200 import _lib
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged, rotary

    rng = np.random.default_rng(7)
    page, hk, h, d, total = 64, 8, 16, 64, 70000
    size = page * hk * d
    keys, values = DeviceArray((total, page, hk, d), "bfloat16"), DeviceArray((total, page, hk, d), "bfloat16")
    q, k0, v0, cu, lens, table = build(rng, [150], [count], h, hk, d, page, False, "bfloat16")
    far = table.copy()
    far[0, :3] = [69999, 65536, 66001]
    for pool, src in ((keys, k0), (values, v0)):
        for i in range(3):
            part = dev(src[table[0, i]], "bfloat16")
            pool.view(int(far[0, i]) * size, (page, hk, d)).copy_(part)
    out, lse = DeviceArray(q.shape, "bfloat16"), DeviceArray(q.shape[:2], "float32")
    cache = paged.PagedCache(keys, values)
    paged.paged_attention(dev(q, "bfloat16"), cache, dev(cu), dev(lens), dev(far), max_q=count, out=out, lse=lse)
    check_attention(out.numpy(), lse.numpy(), q, k0, v0, cu, lens, table, False, "bfloat16", d ** -0.5)
    qkv = normal(rng, (count, (h + 2 * hk) * d), "bfloat16")
    paged.paged_append(dev(qkv, "bfloat16"), cache, dev(cu), dev(lens), dev(far), heads=h,
                       freqs=dev(rotary.rotary_frequencies(d, 1e6)[0]))
    last = keys.view(66001 * size, (page, hk, d)).numpy(), values.view(66001 * size, (page, hk, d)).numpy()
    _, kk, vv = op.split_heads(qkv.astype(np.float64), h, hk, d)
    want = op.head_forward(kk[-1], None, 149, rotary.rotary_frequencies(d, 1e6)[0], 1.0, False, 0.0)
    assert np.all(np.abs(last[0][21].astype(np.float64) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -17)
    np.testing.assert_array_equal(last[1][21], vv[-1].astype(NP["bfloat16"]))
    _lib.call("mfb_device_sync")


def test_paged_attention_long_single_sequence():
    """One row over a long context: its partials are joined in two levels."""
    require_gpu()
    rng = np.random.default_rng(8)
    for counts, h, hk in (([1], 16, 8), ([2], 2, 1), ([24], 2, 1)):
        a = build(rng, [40001], counts, h, hk, 64, 64, False, "bfloat16")
        got, lse = run_attention(*a, False, "bfloat16", counts[0])
        check_attention(got, lse, *a, False, "bfloat16", 0.125)


@pytest.mark.parametrize("count", [1, 50])
def test_paged_attention_bad_tables_are_recorded(count):
    """Contradicting device arguments are clamped, recorded, and leave the buffers' other rows alone."""
    require_gpu()
    from minifield_training_b200.kernels import paged

    rng = np.random.default_rng(9)
    a = build(rng, [200, 100], [count, count], 4, 2, 64, 16, False, "bfloat16", pad=4, gap=0)
    q, keys, values, cu, lens, table = a
    good, _ = run_attention(*a, False, "bfloat16", count)
    paged.paged_attention_status()
    for bad in (len(keys), -7, 1 << 30):
        t = table.copy()
        t[1, 2] = bad
        got, _ = run_attention(q, keys, values, cu, lens, t, False, "bfloat16", count)
        assert paged.paged_attention_status() == 1001
        np.testing.assert_array_equal(got[:count], good[:count])
        assert np.all(got[2 * count:].astype(np.float32) == 5)
    longer = np.array([10 ** 6, 100], np.int32)
    got, _ = run_attention(q, keys, values, cu, longer, table, False, "bfloat16", count)
    assert paged.paged_attention_status() == 1002
    np.testing.assert_array_equal(got[count:2 * count], good[count:2 * count])
    wild = np.array([0, count, 10 ** 6], np.int32)
    got, _ = run_attention(q, keys, values, wild, lens, table, False, "bfloat16", count)
    assert paged.paged_attention_status() == 1002
    np.testing.assert_array_equal(got[:count], good[:count])


def test_paged_attention_streams_and_graphs():
    """Two streams at once give each its own answer; a captured call follows its buffers and needs its own workspace."""
    require_gpu()
    from minifield_training_b200 import _lib
    from minifield_training_b200.device import DeviceArray, sync
    from minifield_training_b200.kernels import paged

    rng = np.random.default_rng(10)
    streams = []
    for _ in range(2):
        s = ctypes.c_void_p()
        _lib.call("mfb_stream_create", ctypes.byref(s))
        streams.append(s.value)
    try:
        for counts in ([1, 1], [90, 20]):
            work = []
            for _ in range(2):
                a = build(rng, [3000, 700], counts, 16, 8, 64, 16, False, "bfloat16")
                q, keys, values, cu, lens, table = a
                cache = paged.PagedCache(dev(keys, "bfloat16"), dev(values, "bfloat16"))
                args = [dev(q, "bfloat16"), cache, dev(cu), dev(lens), dev(table)]
                ref = DeviceArray(q.shape, "bfloat16")
                paged.paged_attention(*args, max_q=max(counts), out=ref)
                work.append((a, args, ref.numpy(), DeviceArray(q.shape, "bfloat16")))
            sync()
            for _ in range(20):
                for (_, args, _, out), s in zip(work, streams):
                    paged.paged_attention(*args, max_q=max(counts), out=out, stream=s)
            for (_, _, ref, out), s in zip(work, streams):
                np.testing.assert_array_equal(out.numpy(s), ref)
            # Captured on one stream, both graphs with a workspace of their own, replayed side by side.
            graphs = []
            need = paged.paged_attention_workspace_size(sum(counts), 2, max(counts), 16, 8, 64)
            for (_, args, _, out) in work:
                _lib.call("mfb_graph_begin", streams[0])
                with pytest.raises(ValueError, match="its own workspace"):
                    paged.paged_attention(*args, max_q=max(counts), out=out, stream=streams[0])
                ws = DeviceArray((need,), "uint8")
                paged.paged_attention(*args, max_q=max(counts), out=out, stream=streams[0], workspace=ws)
                g = ctypes.c_void_p()
                _lib.call("mfb_graph_end", streams[0], ctypes.byref(g))
                graphs.append((g.value, ws))
            shorter = np.array([2500, 300], np.int32)
            want = []
            for (a, args, _, out) in work:
                dst = args[3]
                _lib.call("mfb_memcpy_h2d", dst.ptr, shorter.ctypes.data, shorter.nbytes, None)
                sync()
                ref = DeviceArray(out.shape, "bfloat16")
                paged.paged_attention(*args, max_q=max(counts), out=ref)
                want.append(ref.numpy())
            for _ in range(10):
                for (g, _), s in zip(graphs, streams):
                    _lib.call("mfb_graph_launch", g, s)
            for (_, _, _, out), s, ref in zip(work, streams, want):
                np.testing.assert_array_equal(out.numpy(s), ref)
            for g, _ in graphs:
                _lib.call("mfb_graph_destroy", g)
    finally:
        for s in streams:
            _lib.call("mfb_stream_destroy", s)


@pytest.mark.parametrize("lens, counts, h, hk, d, page, head_major, dtype, part, interleaved, gains", [
    ([1], [1], 16, 8, 64, 16, False, "bfloat16", 64, False, True),
    ([40, 17, 9, 100], [1, 1, 0, 1], 16, 8, 64, 16, False, "bfloat16", 64, False, True),
    ([300, 33, 64], [150, 33, 1], 6, 2, 128, 32, True, "float16", 64, True, False),
    ([20, 3], [33, 3], 4, 1, 64, 8, False, "float16", 16, False, True),  # tokens before the sequence's start
])
def test_append_then_attend(lens, counts, h, hk, d, page, head_major, dtype, part, interleaved, gains):
    """Append writes q and exactly the new rows of the pages; attention reads what it wrote."""
    require_gpu()
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged, rotary

    rng = np.random.default_rng(sum(lens) + d)
    _, keys, values, cu, lens, table = build(rng, lens, counts, h, hk, d, page, head_major, dtype, junk=3.0)
    n, pad = int(cu[-1]), 2
    qkv = normal(rng, (n + pad, (h + 2 * hk) * d + 8), dtype)
    freqs = rotary.rotary_frequencies(part, 1e4)[0]
    wq, wk = ((1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if gains else None for _ in range(2))
    cache = paged.PagedCache(dev(keys, dtype), dev(values, dtype), head_major=head_major)
    out = DeviceArray.from_numpy(np.full((n + pad, h, d), 5, NP[dtype]), dtype)
    arrays = dev(cu), dev(lens), dev(table)
    got_q = paged.paged_append(dev(qkv, dtype), cache, *arrays, heads=h, freqs=dev(freqs), interleaved=interleaved,
                               q_weight=None if wq is None else dev(wq), k_weight=None if wk is None else dev(wk),
                               eps=1e-5, out=out)
    q, k, v = op.split_heads(qkv.astype(np.float64), h, hk, d)
    want_k, want_v = keys.astype(np.float64), values.astype(np.float64)
    turn = lambda x, w, pos: op.head_forward(x, w, pos, freqs, 1.0, interleaved, 1e-5)  # noqa: E731
    want_q = np.full((n + pad, h, d), 5.0)
    for b in range(len(lens)):
        for i in range(counts[b]):
            t, pos = cu[b] + i, lens[b] - counts[b] + i
            want_q[t] = turn(q[t], wq, pos)
            if pos >= 0:
                for pool, row in ((want_k, turn(k[t], wk, pos)), (want_v, v[t])):
                    view = np.swapaxes(pool, 1, 2) if head_major else pool
                    view[table[b, pos // page], pos % page] = row
    u = U[dtype]
    for got, want in ((got_q.numpy(), want_q), (cache.keys.numpy(), want_k)):
        err = np.abs(got.astype(np.float64) - want)
        assert np.all(err <= u * np.abs(want) + 2.0 ** -18 * np.abs(want).max(-1, keepdims=True))
    np.testing.assert_array_equal(cache.values.numpy(), want_v.astype(NP[dtype]))
    # The attention of the stored values, from the stored values.
    kept = got_q.numpy()
    o, lse = DeviceArray.from_numpy(np.full(kept.shape, 5, NP[dtype]), dtype), dev(np.full(kept.shape[:2], 5.0, np.float32))
    paged.paged_attention(got_q, cache, *arrays, max_q=max(counts), out=o, lse=lse)
    check_attention(o.numpy(), lse.numpy(), kept, cache.keys.numpy(), cache.values.numpy(), cu, lens, table, head_major,
                    dtype, d ** -0.5)


def test_append_drops_tokens_without_a_page():
    require_gpu()
    from minifield_training_b200.kernels import paged, rotary

    rng = np.random.default_rng(12)
    page, hk, h, d = 16, 2, 4, 64
    keys = np.full((4, page, hk, d), 3, NP["bfloat16"])
    cache = paged.PagedCache(dev(keys, "bfloat16"), dev(keys, "bfloat16"))
    table = np.array([[0, -1], [1 << 20, 2], [3, 1]], np.int32)
    lens, cu = np.array([17, 16, 40], np.int32), np.array([0, 2, 4, 12], np.int32)
    qkv = normal(rng, (12, (h + 2 * hk) * d), "bfloat16")
    paged.paged_append(dev(qkv, "bfloat16"), cache, dev(cu), dev(lens), dev(table), heads=h,
                       freqs=dev(rotary.rotary_frequencies(d, 1e4)[0]))
    got = cache.values.numpy()
    v = op.split_heads(qkv.astype(np.float64), h, hk, d)[2].astype(NP["bfloat16"])
    want = keys.copy()
    want[0, 15] = v[0]  # position 15 has a page, 16 has none; row 1's page is outside the pool
    np.testing.assert_array_equal(got, want)  # row 2's positions 32..39 lie behind its table


# ---- logits ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows, vocab, n, k, grammars, dtype", [
    (1, 1, 1, 1, 1, "float32"),
    (1, 65536, 300, 8, 1, "bfloat16"),
    (3, 1000, 50, 3, 0, "float32"),
    (5, 50257, 700, 17, 3, "float16"),
    (2, 33, 5, 0, 2, "bfloat16"),
    (4, 4099, 0, 40, 4, "bfloat16"),
    (7, 128256, 3000, 2047, 7, "bfloat16"),
    (2, 393216, 100, 2, 1, "float32"),
    (6, 777, 0, 0, 2, "float16"),
    (2, 500, 20000, 4, 0, "float32"),
])
def test_logit_controls(rows, vocab, n, k, grammars, dtype):
    require_gpu()
    from minifield_training_b200.kernels import logits as lg

    rng = np.random.default_rng(rows + vocab)
    x = (3 * rng.standard_normal((rows, vocab), dtype=np.float32)).astype(NP[dtype])
    x[0, 0] = -np.inf
    if vocab > 40:
        x[-1, 3], x[-1, 4] = 0.0, np.inf
    kw = {}
    if n:
        hist = rng.integers(-2, max(vocab // 3, 1) + 2, (rows, n)).astype(np.int32)
        hist[:, : n // 2] = hist[:, n // 2: 2 * (n // 2)]  # every token at least twice
        hist[0, -1] = vocab  # outside
        used = rng.integers(0, n + 1, rows).astype(np.int32)
        used[0] = n + 7 if rows > 1 else n  # clamped
        kw.update(history=hist, history_len=used, prompt_len=(used * rng.random(rows)).astype(np.int32),
                  repetition=(1 + rng.random(rows)).astype(np.float32), frequency=rng.random(rows).astype(np.float32),
                  presence=rng.standard_normal(rows).astype(np.float32))
    if k:
        ids = rng.integers(-1, vocab + 1, (rows, k)).astype(np.int32)
        ids[:, -1] = ids[:, 0]  # the same index twice: the last counts
        kw.update(bias_ids=ids, bias_values=rng.standard_normal((rows, k)).astype(np.float32))
    if grammars:
        kw["mask"] = rng.integers(-(1 << 31), 1 << 31, (grammars, (vocab + 31) // 32)).astype(np.int32)
        kw["mask"][0] = 0  # a grammar that allows nothing
        if grammars < rows or rows % 2:
            kw["mask_rows"] = rng.integers(-1, grammars + 1, rows).astype(np.int32)
    got = lg.process_logits(dev(x, dtype), **{a: dev(b) for a, b in kw.items()}).numpy()
    want = op.controlled_logits(x.astype(np.float64), **kw)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin].astype(np.float32))
    # Four FP32 operations, each at most half a step of the largest term.
    size = np.abs(x.astype(np.float64)) * (kw["repetition"][:, None] if n else 1.0)
    terms = (kw["frequency"][:, None] * n + np.abs(kw["presence"][:, None])) if n else 0.0
    bias = 6.0 if k else 0.0
    bound = 4 * 2.0 ** -24 * np.broadcast_to(np.where(np.isfinite(size), size, 0) + terms + bias, x.shape)
    assert np.all(np.abs(got.astype(np.float64)[fin] - want[fin]) <= bound[fin])
    if not n and not k:
        np.testing.assert_array_equal(got[fin], x.astype(np.float32)[fin])


def test_logits_in_place_and_defaults():
    require_gpu()
    from minifield_training_b200.kernels import logits as lg

    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 999), dtype=np.float32)
    hist = rng.integers(0, 999, (3, 64)).astype(np.int32)
    f = rng.random(3).astype(np.float32)
    a = dev(x)
    out = lg.process_logits(a, history=dev(hist), frequency=dev(f), out=a)
    assert out is a
    want = op.controlled_logits(x, history=hist, frequency=f)
    assert np.all(np.abs(a.numpy() - want) <= 2.0 ** -23 * (np.abs(x) + 64 * f[:, None]))
    np.testing.assert_array_equal(lg.process_logits(dev(x)).numpy(), x)
