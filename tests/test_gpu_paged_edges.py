"""Edges of the rotary, paged-cache and logit operators on the GPU: the largest sizes, many items, odd values.

Helpers and tolerances are those of tests/test_gpu_paged.py.
"""

import ctypes

import numpy as np
import pytest

from oracle import paged as op
from tests.gpu_env import require_gpu
from tests.test_gpu_paged import NP, U, build, check_attention, dev, normal, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [1, 20])
def test_sequence_that_ends_just_below_2_31(count):
    """The look-ahead of page ids (4096 keys) passes 2^31; every page of the table is the pool's one page.

    Keys are zeros, so all weights are equal, and the values are 1/2. A row part's sums of n <= 2^31 / 148 ones and
    halves are exact in FP32 but for the polynomial exponential (2.7e-6), the joins round at most 300 times by
    2^-24: below 2^-15 in all, where half a step of bf16 under 1/2 is 2^-10.
    """
    require_gpu()
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged

    page, pages = 1024, (1 << 21) - 1
    length = page * pages - 5
    keys, values = np.zeros((1, page, 1, 64), NP["bfloat16"]), np.full((1, page, 1, 64), 0.5, NP["bfloat16"])
    cache = paged.PagedCache(dev(keys, "bfloat16"), dev(values, "bfloat16"))
    q = dev(np.ones((count, 1, 64), NP["bfloat16"]), "bfloat16")
    lse = DeviceArray((count, 1), "float32")
    paged.paged_attention_status()
    out = paged.paged_attention(q, cache, dev(np.array([0, count], np.int32)), dev(np.array([length], np.int32)),
                                dev(np.zeros((1, pages), np.int32)), max_q=count, lse=lse)
    got = out.numpy().astype(np.float32)
    assert paged.paged_attention_status() == 0
    np.testing.assert_array_equal(got, 0.5)
    want = np.log(length - count + 1.0 + np.arange(count))
    assert np.all(np.abs(lse.numpy()[:, 0] - want) <= 2.0 ** -18 * want)


def test_sequences_that_claim_the_same_rows_past_2_31_items():
    """cu_q = 0, N, 0, N, ...: 4096 sequences of all N rows each, 2^31 items in all, are counted and cut at the list."""
    require_gpu()
    from minifield_training_b200 import _lib
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged

    n, batch = 1 << 27, 8192
    q = DeviceArray((n, 1, 64), "bfloat16")
    _lib.call("mfb_memset", q.ptr, 0x40, q.nbytes, None)  # 0x4040: 3.0
    pool = np.full((1, 16, 1, 64), 1.5, NP["bfloat16"])
    cache = paged.PagedCache(dev(pool, "bfloat16"), dev(pool, "bfloat16"))
    cu = np.zeros(batch + 1, np.int32)
    cu[1::2] = n
    paged.paged_attention_status()
    paged.paged_attention(q, cache, dev(cu), dev(np.ones(batch, np.int32)), dev(np.zeros((batch, 1), np.int32)),
                          max_q=n, out=q)
    assert paged.paged_attention_status() == 1002
    for at in (0, 1 << 26, n - 1001):  # a sequence's only token is its last row's key
        assert not np.any(q.view(at * 64, (1000, 64)).numpy().astype(np.float32))
    np.testing.assert_array_equal(q.view((n - 1) * 64, (64,)).numpy().astype(np.float32), 1.5)


def test_streams_have_identities_of_their_own():
    """Handles come again after a stream is destroyed, identities do not; the default stream keeps its own."""
    require_gpu()
    from minifield_training_b200 import _lib

    identity = _lib.stream_identity
    default = identity(None)
    assert default >> 48 == 1  # device 0
    seen, word = {default}, dev(np.zeros(1, np.int32))
    for _ in range(20):
        s = ctypes.c_void_p()
        _lib.call("mfb_stream_create", ctypes.byref(s))
        assert identity(s.value) not in seen and identity(s.value) == identity(s.value)
        seen.add(identity(s.value))
        _lib.call("mfb_graph_begin", s.value)
        assert identity(s.value) == 0 and identity(None) == default
        _lib.call("mfb_memset", word.ptr, 0, 4, s.value)
        g = ctypes.c_void_p()
        _lib.call("mfb_graph_end", s.value, ctypes.byref(g))
        _lib.call("mfb_graph_destroy", g.value)
        _lib.call("mfb_stream_destroy", s.value)
    assert len(seen) == 21 and identity(None) == default == identity(ctypes.c_void_p(1))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_infinite_penalties_reach_only_their_tokens(dtype):
    """A token that was not generated keeps its logit, beside generated ones as anywhere else."""
    require_gpu()
    from minifield_training_b200.kernels import logits as lg

    rng = np.random.default_rng(14)
    x = rng.standard_normal((3, 100), dtype=np.float32).astype(NP[dtype])
    hist = np.array([[40, 8, 9, 9, 63], [0, 99, 99, 1, 98], [7, 7, 7, 7, 7]], np.int32)
    inf = np.float32(np.inf)
    for name, values in (("frequency", [inf, inf, -inf]), ("presence", [inf, -inf, inf])):
        kw = dict(history=hist, prompt_len=np.array([1, 1, 0], np.int32), **{name: np.array(values, np.float32)})
        got = lg.process_logits(dev(x, dtype), **{k: dev(v) for k, v in kw.items()}).numpy()
        np.testing.assert_array_equal(got, op.controlled_logits(x, **kw).astype(np.float32))


@pytest.mark.parametrize("lens, counts, h, hk, dtype", [
    ([70, 9], [1, 1], 16, 8, "bfloat16"),  # whole items
    ([9000, 40], [2, 1], 4, 2, "float16"),  # items cut between CTAs
    ([300, 64], [40, 64], 4, 2, "bfloat16"),  # tiles
    ([9000, 300], [200, 30], 2, 1, "float16"),  # tiles, cut
])
def test_queries_that_are_not_numbers(lens, counts, h, hk, dtype):
    """A NaN query gives NaN in its output and its lse, not the -inf of a token without keys; the others see nothing."""
    require_gpu()
    rng = np.random.default_rng(15)
    a = build(rng, lens, counts, h, hk, 64, 16, False, dtype, pad=2)
    good, good_lse = run_attention(*a, False, dtype, max(counts))
    q, hurt = a[0].copy(), np.zeros(a[0].shape[:2], bool)
    for t, head in ((0, 0), (int(a[3][1]) - 1, 1), (int(a[3][2]) - 1, h - 1)):
        q[t, head, 5], hurt[t, head] = np.nan, True
    got, lse = run_attention(q, *a[1:], False, dtype, max(counts))
    np.testing.assert_array_equal(got[~hurt], good[~hurt])
    np.testing.assert_array_equal(lse[~hurt], good_lse[~hurt])
    assert np.all(np.isnan(got[hurt].astype(np.float32))) and np.all(np.isnan(lse[hurt]))


def test_gradient_of_columns_behind_the_heads():
    """Zeros in a new array, over memory that held something else."""
    require_gpu()
    from minifield_training_b200 import _lib
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import rotary

    rng = np.random.default_rng(16)
    qkv, grads = normal(rng, (50, 2048 + 24), "bfloat16"), [normal(rng, (50, n, 64), "bfloat16") for n in (16, 8, 8)]
    freqs, pos = dev(rotary.rotary_frequencies(64, 1e4)[0]), dev(np.arange(50, dtype=np.int32))
    args = [dev(qkv, "bfloat16"), pos, freqs, *(dev(g, "bfloat16") for g in grads)]
    for _ in range(3):
        old = DeviceArray(qkv.shape, "bfloat16")
        _lib.call("mfb_memset", old.ptr, 0x40, old.nbytes, None)
        _lib.call("mfb_device_sync")
        del old  # its memory is the likely place of the next array of this size
        got = rotary.qk_rotary_bwd(*args, head_dim=64)[0].numpy()
        assert not np.any(got[:, 2048:].astype(np.float32)) and np.all(np.any(got[:, :2048], 1))


@pytest.mark.parametrize("batch, counts, h, hk, page, dtype", [
    (1300, (0, 1, 1, 2), 4, 2, 8, "bfloat16"),  # few rows: several items per thread of a CTA's own schedule
    (700, (1,), 6, 3, 16, "float16"),  # three head groups per sequence
    (1500, (0, 1, 3, 20), 2, 1, 16, "bfloat16"),  # tiles: more sequences and items than the schedule kernel has threads
    (131, (129,), 8, 4, 64, "float16"),  # two query blocks per head: 1048 items
])
def test_more_items_and_sequences_than_threads(batch, counts, h, hk, page, dtype):
    """Against float64, and bit for bit the same again (cut items are joined in share order)."""
    require_gpu()
    from minifield_training_b200.kernels import paged

    rng = np.random.default_rng(batch)
    count = rng.choice(counts, batch)
    lens = count + rng.integers(0, 40, batch) - rng.integers(0, 2, batch) * (count > 1)
    lens[rng.integers(0, batch, 3)] += 2500  # long ones are cut between CTAs
    a = build(rng, [int(n) for n in lens], [int(n) for n in count], h, hk, 64, page, False, dtype, pad=3)
    paged.paged_attention_status()
    got, lse = run_attention(*a, False, dtype, max(counts))
    assert paged.paged_attention_status() == 0
    check_attention(got, lse, *a, False, dtype, 0.125)
    again, lse2 = run_attention(*a, False, dtype, max(counts))
    np.testing.assert_array_equal(again.view(np.uint16), got.view(np.uint16))
    np.testing.assert_array_equal(lse2, lse)


@pytest.mark.parametrize("lens, counts, h, hk, page, head_major, dtype", [
    ([147, 2013, 420, 671, 1800, 2692, 908, 1609], [27, 27, 8, 32, 1, 12, 22, 14], 40, 8, 32, True, "bfloat16"),
    ([2680, 2794, 677, 609, 2711, 984], [4, 2, 6, 3, 6, 1], 48, 3, 8, True, "float16"),
    ([72, 2645, 5, 2196, 1545, 1927, 341, 1859, 2436], [4, 5, 3, 1, 5, 4, 5, 3, 20], 2, 1, 8, False, "float16"),
    ([545, 365, 155, 75, 448, 656, 109, 434, 582, 643, 702], [2, 2, 0, 2, 2, 2, 0, 3, 3, 1, 3], 7, 1, 8, False, "bfloat16"),
])
def test_tiles_whose_values_come_late(lens, counts, h, hk, page, head_major, dtype):
    """Many small boxes per tile: an item's last softmax may end before the product of the tile before it starts.

    The outputs are read only behind both; every one of many calls, back to back, gives the same bits.
    """
    require_gpu()
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels import paged

    rng = np.random.default_rng(sum(lens) + h + 64)
    a = build(rng, lens, counts, h, hk, 64, page, head_major, dtype)
    q, keys, values, cu, n, table = a
    first, lse = run_attention(*a, head_major, dtype, max(counts))
    check_attention(first, lse, *a, head_major, dtype, 0.125)
    cache = paged.PagedCache(dev(keys, dtype), dev(values, dtype), head_major=head_major)
    args = [dev(q, dtype), cache, dev(cu), dev(n), dev(table)]
    outs = [DeviceArray(q.shape, dtype) for _ in range(10)]
    for _ in range(20):
        for out in outs:
            paged.paged_attention(*args, max_q=max(counts), out=out)
        for out in outs:
            np.testing.assert_array_equal(out.numpy().view(np.uint16), first.view(np.uint16))
    assert paged.paged_attention_status() == 0
