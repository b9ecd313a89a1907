"""Host side of the rotary, paged-cache and logit operators at their edges (no GPU): a library that only records its calls."""

import ctypes
import dataclasses
import math
import threading

import numpy as np
import pytest

from minifield_training_b200 import _lib, device
from minifield_training_b200.device import DeviceArray
from minifield_training_b200.kernels import paged, rotary


class FakeDevice:
    """Answers the runtime calls: memory is a counter, streams have the ids given to them, nothing else runs."""

    def __init__(self):
        self.calls, self.packed, self.next, self.live = [], [], 1 << 20, {}
        self.current, self.ids, self.capturing = 0, {}, set()

    def call(self, name, *args):
        self.calls.append((name, args))
        if name == "mfb_paged_attn_check":  # arithmetic on the host
            _lib.check(getattr(_lib.lib(), name)(*args), name)
        if name == "mfb_malloc":
            args[0]._obj.value = self.next
            self.live[self.next] = int(args[1])
            self.next += -(-int(args[1]) // 256) * 256
        elif name == "mfb_graph_end":
            args[1]._obj.value = 1

    def stream_identity(self, stream):
        handle = getattr(stream, "value", stream)
        number = self.ids.get((self.current, handle), handle or 1)
        return 0 if handle in self.capturing else (self.current + 1 << 48) + number

    def call_packed(self, name, flags, *args, stream=None):
        self.packed.append((name, args))

    def names(self):
        return [name for name, _ in self.calls]


@pytest.fixture
def fake(monkeypatch):
    f = FakeDevice()
    monkeypatch.setattr(_lib, "call", f.call)
    monkeypatch.setattr(_lib, "call_packed", f.call_packed)
    monkeypatch.setattr(_lib, "stream_identity", f.stream_identity)
    monkeypatch.setattr(DeviceArray, "__del__", lambda self: f.live.pop(self.ptr) if self._owner else None)
    monkeypatch.setattr(device, "_STREAM_WORKSPACES", {})
    return f


def array(shape, dtype, ptr=1 << 20):
    return DeviceArray(shape, dtype, ptr=ptr, owner=False)


def test_stream_workspaces_are_kept_per_device_stream_and_thread(fake):
    def get(stream=None, nbytes=1000):
        return device.stream_workspace("w", nbytes, stream)

    first = get()
    assert get() is first and get(stream=0) is first and get(stream=ctypes.c_void_p(1)) is first  # one stream
    assert get(stream=64) is not first
    fake.current = 1
    other = get()  # the default stream's handle is the same on every device
    assert other is not first and get() is other and get(stream=64) is not other
    fake.current = 0
    assert get() is first
    mine, theirs = get(stream=2), []
    thread = threading.Thread(target=lambda: theirs.append(get(stream=2)))
    thread.start()
    thread.join()
    assert get(stream=2) is mine and theirs[0] is not mine


def test_a_reused_stream_handle_gets_a_new_workspace(fake):
    old = device.stream_workspace("w", 1000, 64)
    fake.ids[0, 64] = 7  # the handle's stream was destroyed (its work may still run), a new one has the handle
    new = device.stream_workspace("w", 1000, 64)
    assert new is not old and device.stream_workspace("w", 1000, 64) is new
    fake.capturing.add(64)
    for nbytes in (10, 5000):
        with pytest.raises(ValueError, match="its own workspace"):
            device.stream_workspace("w", nbytes, 64)


@pytest.mark.parametrize("length, factor, low, high", [(4096, 16, 10, 23), (65536, 4, 20, 33), (131072, 8, 22, 35)])
def test_yarn_divides_only_pairs_that_turn_too_seldom(length, factor, low, high):
    """Rotary 64, theta 1e4: pair i turns length 1e4^(-i / 32) / 2 pi times, 32 and once at the bounds given here.

    The ramp runs between the whole pairs around those bounds, also where the second one lies behind the last pair.
    """
    index = np.arange(32)
    base = 1e4 ** (-index / 32.0)
    turns = length * base / (2 * math.pi)
    pair = [32 * math.log(length / (t * 2 * math.pi)) / math.log(1e4) for t in (32.0, 1.0)]
    assert (math.floor(pair[0]), math.ceil(pair[1])) == (low, high)
    share = np.array([min(max((i - low) / (high - low), 0.0), 1.0) for i in index])  # of the divided frequency
    got = rotary.rotary_frequencies(64, 1e4, {"kind": "yarn", "factor": factor, "original_length": length})[0]
    np.testing.assert_allclose(got, base * ((1 - share) + share / factor), rtol=2.0 ** -22)
    assert np.all(got[turns > 1.0] > base[turns > 1.0] / factor * (1 + 2.0 ** -20))


@pytest.mark.parametrize("pages, columns", [(0, 5), (9, 0), (0, 0)])
def test_append_and_attention_refuse_a_cache_without_pages(pages, columns):
    """Both refuse; append once returned a q that nothing had written."""
    cache = paged.PagedCache(*[array((pages, 16, 8, 64), "bfloat16")] * 2)
    cu, lens, table = array((3,), "int32"), array((2,), "int32"), array((2, columns), "int32")
    q = array((4, 16, 64), "bfloat16")
    with pytest.raises(ValueError, match="pages"):
        paged.paged_append(array((4, 2048), "bfloat16"), cache, cu, lens, table, heads=16,
                           freqs=array((32,), "float32"), out=q)
    with pytest.raises(ValueError, match="pages"):
        paged.paged_attention(q, cache, cu, lens, table, max_q=2, out=q, workspace=array((1 << 30,), "uint8"))


@pytest.mark.parametrize("which", [0, 1])
def test_rotary_backward_adds_only_to_given_gradients(fake, which):
    """A missing one of the two is a new array, which holds nothing that could be added to."""
    qkv, w = array((4, 2048), "bfloat16"), array((64,), "float32")
    args = [qkv, array((4,), "int32"), array((32,), "float32"), array((4, 16, 64), "bfloat16"),
            array((4, 8, 64), "bfloat16"), array((4, 8, 64), "bfloat16")]
    grads = [w, w]
    grads[which] = None
    with pytest.raises(ValueError, match="to add to"):
        rotary.qk_rotary_bwd(*args, q_weight=w, k_weight=w, weight_grads=tuple(grads), accumulate=True)
    got = rotary.qk_rotary_bwd(*args, q_weight=w, k_weight=w, weight_grads=tuple(grads))[1:]
    assert got[1 - which] is w and got[which] is not w and got[which].shape == (64,)


@pytest.mark.parametrize("extra", [0, 8])
def test_rotary_backward_clears_columns_without_heads(fake, extra):
    """A projection may be wider than its heads: the gradient of the rest is zero, in a new array or as given."""
    qkv, out = array((4, 2048 + extra), "bfloat16"), array((4, 2048 + extra), "bfloat16")
    args = [qkv, array((4,), "int32"), array((32,), "float32"), array((4, 16, 64), "bfloat16"),
            array((4, 8, 64), "bfloat16"), array((4, 8, 64), "bfloat16")]
    rotary.qk_rotary_bwd(*args, head_dim=64, out=out, stream=64)
    assert "mfb_memset" not in fake.names()
    dqkv = rotary.qk_rotary_bwd(*args, head_dim=64, stream=64)[0]
    cleared = [a for name, a in fake.calls if name == "mfb_memset"]
    assert cleared == ([(dqkv.ptr, 0, 4 * 2056 * 2, 64)] if extra else [])
    assert [name for name, _ in fake.packed] == ["mfb_qk_rotary_bwd"] * 2


def test_a_new_cache_is_clear_before_any_stream_uses_it(fake):
    """The clearing runs on the default stream, which created streams do not wait for."""
    cache = paged.PagedCache.zeros(9, 16, 8, 64)
    assert fake.names()[-3:] == ["mfb_malloc", "mfb_memset", "mfb_stream_sync"]
    assert [a[0].value for name, a in fake.calls if name == "mfb_memset"] == [cache.keys.ptr, cache.values.ptr]
    assert fake.calls[-1][1] == (None,)


def decoder(stream=None, **changes):
    """A decoder (conv, attention, conv, attention) on the recorded library, and its config."""
    from minifield_training_b200 import workloads
    from minifield_training_b200.models import decode
    cfg = dataclasses.replace(workloads.DECODER, **{**dict(
        hidden=256, ffn=512, heads=4, kv_heads=2, vocab=1000,
        layer_types=("conv", "full_attention", "conv", "full_attention")), **changes})
    return decode.Decoder(cfg, decode.init_parameters(cfg, 0), stream=stream), cfg, decode


def test_extend_refuses_before_anything_runs(fake):
    dec, cfg, dm = decoder(max_position_embeddings=1 << 26)
    state = dm.new_paged_state(cfg, 1, 1 << 20, 64)
    dec.extend(np.zeros((1, 5), np.int32), state)
    before = list(state.lengths), state.table.copy(), list(state._free), len(fake.packed)
    ids = np.zeros((1, 3), np.int32)
    wide = array((1, cfg.vocab), "float32", ptr=(1 << 20) + 4)
    for match, call in (
            ("2.31 key tiles", lambda: dec.extend(np.zeros((1, 1 << 18), np.int32), state)),
            ("16-byte aligned", lambda: dec.extend(ids, state, out=wide)),
            ("device array", lambda: dec.extend(ids, state, out=np.zeros((1, cfg.vocab), np.float32)))):
        with pytest.raises(ValueError, match=match):
            call()
        assert (list(state.lengths), list(state._free), len(fake.packed)) == (before[0], before[2], before[3])
        assert np.array_equal(state.table, before[1])
    state = dm.new_paged_state(cfg, 2, 4, 1 << 24)  # a page of 2^31 elements is more than the kernels take
    with pytest.raises(ValueError, match="too large"):
        dec.extend(np.zeros((2, 1), np.int32), state)
    assert state.lengths == [0, 0] and len(state._free) == 4


def test_a_step_uploads_its_tokens_and_the_pages_it_took(fake):
    """Not the whole table, however wide; rows are no wider than the model's positions."""
    dec, cfg, dm = decoder(max_position_embeddings=6400)
    state = dm.new_paged_state(cfg, 4, 1 << 16, 64)
    assert state.max_pages == 100 and dm.new_paged_state(cfg, 4, 30, 64).max_pages == 30

    def uploads(call):
        start = len(fake.calls)
        call()
        return [(a[0].value, a[2]) for name, a in fake.calls[start:] if name == "mfb_memcpy_h2d"]

    def step(t, rows=None):
        return uploads(lambda: dec.extend(np.zeros((len(rows or range(4)), t), np.int32), state, rows=rows))

    at = state.device_table.ptr
    assert step(130)[1:] == [(at + 400 * row, 12) for row in range(4)]  # three pages each
    first = step(1)
    assert len(first) == 1 and first[0][1] == 4 * (4 + 5 + 4)  # tokens, offsets, lengths
    step(60, range(1, 2))
    assert step(2, range(1, 2))[1:] == [(at + 400 + 12, 4)]  # the 193rd token's page
    assert at + 400 in fake.packed[-1][1]  # attention reads the rows' part of the table in place
    state.release(1)
    assert step(1, range(1, 2))[1:] == [(at + 400, 4)]
    state.grow(range(2, 3), 126)  # 131 tokens before, 257 now: pages 3 and 4
    assert uploads(lambda: state.upload(5)) == [(at + 800 + 12, 8)] and uploads(state.upload) == []


def test_scratch_of_extend_is_bounded(fake):
    """One set for all calls, as large as the largest needed, and one per power of two of rows for captured steps."""
    dec, cfg, dm = decoder(stream=64)
    state = dm.new_paged_state(cfg, 64, 64 * 80, 64)
    rng = np.random.default_rng(17)

    def call(b, t, graph=False):
        for row in range(b):
            state.release(row)
        dec.extend(np.zeros((b, t), np.int32), state, rows=range(b), graph=graph)
        return sum(fake.live.values())

    start = sum(fake.live.values())
    largest = call(64, 512) - start
    dec.close()
    assert sum(fake.live.values()) == start
    for b, t in [(int(b), int(t)) for b, t in zip(rng.integers(1, 65, 60), 2 ** rng.integers(0, 9, 60))]:
        assert call(b, t) - start <= largest
    assert call(64, 512) - start == largest
    for b in range(1, 65):
        call(b, 1, graph=True)
    assert len(dec._extend_scratch) == 1 + 7
    kept = {id(B): {k: getattr(v, "ptr", v) for k, v in B.items()} for B in dec._extend_scratch.values()}
    for b in (64, 3, 17):
        call(b, 1, graph=True)  # a captured step's buffers stay where they are
    assert kept == {id(B): {k: getattr(v, "ptr", v) for k, v in B.items()} for B in dec._extend_scratch.values()}
    dec._graphs.clear()  # handles of the recorded library
    dec.close()
    assert sum(fake.live.values()) == start
    for b, t in ((33, 512), (1, 1000), (64, 17), (7, 1)):
        dec.close()
        call(b, t)
        B = dec._extend_scratch[None]
        assert b * t <= B["tokens"] <= 1.125 * b * t and b <= B["rows"] <= 1.125 * b


def test_neighbouring_fresh_rows_are_cleared_together(fake):
    dec, cfg, dm = decoder()
    state = dm.new_paged_state(cfg, 8, 64, 64)
    row = 2 * 256 * 2  # bytes of a row's two conv inputs
    layers = [h.ptr for h in state.history if h is not None]

    def cleared(rows):
        start = len(fake.calls)
        dec.extend(np.zeros((len(rows), 3), np.int32), state, rows=rows)
        return [(a[0].value, a[2]) for name, a in fake.calls[start:] if name == "mfb_memset"]

    assert cleared(range(0, 8)) == [(p, 8 * row) for p in layers]
    assert cleared(range(0, 8)) == []
    for r in (1, 2, 5, 7):
        state.release(r)
    assert cleared(range(1, 7)) == [(p + r * row, n * row) for p in layers for r, n in ((1, 2), (5, 1))]


def test_a_captured_step_with_controls_widens_its_logits_once(fake):
    dec, cfg, dm = decoder(stream=64)
    state, ids = dm.new_state(cfg, 2, 16), np.zeros(2, np.int32)
    bias = dict(bias_ids=array((2, 1), "int32"), bias_values=array((2, 1), "float32"))
    done = []
    for controls in (None, bias, bias, None):
        start = len(fake.calls), len(fake.packed)
        dec.decode_one(ids, state, graph=True, controls=controls)
        names = [name for name, _ in fake.calls[start[0]:]]
        done.append((names.count("mfb_cast_bf16_f32"), names.count("mfb_graph_begin"),
                     [name for name, _ in fake.packed[start[1]:]]))
    dec._graphs.clear()  # handles of the recorded library
    controlled = ["mfb_logits_process"]
    assert done == [(1, 1, []), (0, 1, controlled), (0, 0, controlled), (0, 0, [])]


@pytest.mark.parametrize("rows, tokens", [((0, 0), 10), ((-1,), 3), ((2,), 3), ((0,), 0), ((1,), -2)])
def test_pages_go_to_distinct_rows(fake, rows, tokens):
    """The pages of a row named twice were counted from its first length both times: fewer than its tokens need."""
    _, cfg, dm = decoder()
    state = dm.new_paged_state(cfg, 2, 8, 8)
    state.grow((0, 1), 5)
    with pytest.raises(ValueError, match="distinct rows"):
        state.grow(rows, tokens)
    assert state.lengths == [5, 5] and len(state._free) == 6


def test_graphs_of_a_state_that_is_gone_are_released(fake):
    """Behind a synchronise of the stream, by the next captured or replayed step; a living state's stay."""
    dec, cfg, dm = decoder(stream=64)

    def step(state, rows=None):
        start = len(fake.calls)
        dec.extend(np.zeros((len(rows or range(2)), 1), np.int32), state, rows=rows, graph=True)
        return [n for n in fake.names()[start:] if n in ("mfb_stream_sync", "mfb_graph_destroy", "mfb_graph_end")]

    kept = dm.new_paged_state(cfg, 2, 8, 64)
    for _ in range(5):
        state = dm.new_paged_state(cfg, 2, 8, 64)
        assert step(state)[-1:] == step(state, range(1, 2)) == ["mfb_graph_end"]
        del state
    assert step(kept) == ["mfb_stream_sync"] + 2 * ["mfb_graph_destroy"] + ["mfb_graph_end"]
    assert step(kept) == [] and len(dec._graphs) == 1
    dec._graphs.clear()  # handles of the recorded library
