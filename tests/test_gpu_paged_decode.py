"""Decoding over a paged state (models.decode.Decoder.extend) against oracle/decode_model.py.

The decoder of the cached tests (conv, attention, conv, attention; hidden 256,
4/2 heads). ``extend`` rounds the rotated queries and keys, the probabilities
and the outputs once where the oracle rounds step by step, and one rounding that
falls the other way changes all later ones: the two agree as two evaluations
with roundings of their own. A bf16 rounding has an rms error of 2^-7 / sqrt(12)
of the binade's base, 0.7 of that of a value spread over the binade: 1.6e-3. Some
15 roundings a block (two norms, five products, gate, activation, residual sums)
in four blocks give sqrt(60) * 1.6e-3 = 1.2e-2 of rel-L2 against unrounded
logits (the oracle run without its roundings differs from itself by 0.9e-2 to
1.5e-2 per row), and sqrt(2) times that, 1.8e-2, between two evaluations: 2e-2
here. The largest of some thousand errors is four to five sigma, with logits of
rms 0.4 below 4e-2 of the unit of one. A lost or misplaced token moves logits by
tens of percent.
"""

import numpy as np
import pytest

from tests.gpu_env import require_gpu
from tests.test_gpu_decode_model import _cfg

pytestmark = pytest.mark.gpu


def _close(got, ref, what):
    unit = np.maximum(1.0, np.abs(ref))
    err, rel = np.max(np.abs(got - ref) / unit), np.linalg.norm(got - ref) / np.linalg.norm(ref)
    assert err <= 4e-2 and rel <= 2e-2, (what, err, rel)


class Row:
    """One row's tokens through the oracle: prefill of the first chunk, then token by token."""

    def __init__(self, cfg, params, capacity=96):
        self.cfg, self.params, self.capacity, self.state = cfg, params, capacity, None

    def feed(self, ids):
        from oracle import decode_model as odm
        ids = np.asarray(ids, np.int32).reshape(1, -1)
        if self.state is None:
            logits, self.state = odm.prefill(self.cfg, self.params, ids, self.capacity)
            return logits
        for t in ids[0]:
            logits, self.state = odm.decode_one(self.cfg, self.params, np.array([t], np.int32), self.state)
        return logits


@pytest.fixture(scope="module")
def model():
    require_gpu()
    from minifield_training_b200.models import decode as dm
    cfg = _cfg()
    params = dm.init_parameters(cfg, 0)
    return dm, cfg, params, dm.Decoder(cfg, params)


def _feed(model, state, oracles, rows, ids):
    dec = model[3]
    got = dec.extend(ids, state, rows=rows).numpy()
    assert got.shape == (len(ids), model[1].vocab) and got.dtype == np.float32
    for j, r in enumerate(rows if rows is not None else range(state.batch)):
        _close(got[j:j + 1], oracles[r].feed(ids[j]), f"row {r} at {state.lengths[r]}")


@pytest.mark.parametrize("page_size, chunks", [(8, (20, 1, 16, 1, 1)), (64, (37, 1, 1, 30)), (16, (1, 1, 1, 1)),
                                               (16, (2, 3))])
def test_chunks_and_single_tokens_match_the_oracle(model, page_size, chunks):
    dm, cfg, params, _ = model
    state = dm.new_paged_state(cfg, 3, 40, page_size)
    oracles = [Row(cfg, params) for _ in range(3)]
    rng = np.random.default_rng(page_size + sum(chunks))
    for t in chunks:
        _feed(model, state, oracles, None, rng.integers(0, cfg.vocab, (3, t)).astype(np.int32))
    assert state.lengths == [sum(chunks)] * 3


def test_rows_of_their_own_lengths_and_pages_used_again(model):
    dm, cfg, params, _ = model
    state = dm.new_paged_state(cfg, 4, 12, 8)
    oracles = [Row(cfg, params) for _ in range(4)]
    rng = np.random.default_rng(7)

    def ids(n, t):
        return rng.integers(0, cfg.vocab, (n, t)).astype(np.int32)

    _feed(model, state, oracles, range(0, 1), ids(1, 21))
    _feed(model, state, oracles, range(1, 4), ids(3, 5))
    _feed(model, state, oracles, range(2, 4), ids(2, 6))
    for _ in range(2):
        _feed(model, state, oracles, None, ids(4, 1))
    assert state.lengths == [23, 7, 13, 13]
    free = len(state._free)
    held = set(state.table[0, :3])
    state.release(0)
    assert len(state._free) == free + 3 and state.lengths[0] == 0
    oracles[0] = Row(cfg, params)
    _feed(model, state, oracles, range(0, 1), ids(1, 9))  # over the pages row 0 gave back
    assert set(state.table[0, :2]) <= held
    state.release(2)
    oracles[2] = Row(cfg, params)
    for _ in range(3):  # row 2 starts anew with single tokens
        _feed(model, state, oracles, None, ids(4, 1))
    assert state.lengths == [12, 10, 3, 16]
    used = [int(p) for r in range(4) for p in state.table[r] if p >= 0]
    assert len(set(used)) == len(used) and set(used).isdisjoint(state._free)


def test_refusals_leave_the_state_as_it_was(model):
    dm, cfg, params, dec = model
    state = dm.new_paged_state(cfg, 2, 3, 8, max_pages=2)
    oracles = [Row(cfg, params) for _ in range(2)]
    rng = np.random.default_rng(9)
    _feed(model, state, oracles, None, rng.integers(0, cfg.vocab, (2, 7)).astype(np.int32))
    before = (list(state.lengths), state.table.copy(), list(state._free))
    two = np.zeros((2, 2), np.int32)
    for error, call in (
            (dm.DecodeOverflow, lambda: dec.extend(two, state)),  # two more pages, one is free
            (dm.DecodeOverflow, lambda: dec.extend(np.zeros((1, 10), np.int32), state, rows=range(1))),  # three pages
            (ValueError, lambda: dec.extend(two[:1], state)),
            (ValueError, lambda: dec.extend(two, state, rows=range(1, 3))),
            (ValueError, lambda: dec.extend(two, state, controls=dict(history=np.zeros((3, 4), np.int32)))),
            (TypeError, lambda: dec.extend(two, state, controls=dict(temperature=1)))):
        with pytest.raises(error):
            call()
    assert (list(state.lengths), list(state._free)) == (before[0], before[2])
    assert np.array_equal(state.table, before[1])
    _feed(model, state, oracles, range(1, 2), np.array([[3, 4]], np.int32))


def test_single_tokens_replayed_as_a_graph(model):
    """The captured step reads lengths, pages and tokens anew: bit-equal to the launched one, pages taken between."""
    import ctypes
    from minifield_training_b200 import _lib
    dm, cfg, params, plain = model
    stream = ctypes.c_void_p()
    _lib.call("mfb_stream_create", ctypes.byref(stream))
    dec = dm.Decoder(cfg, params, stream=stream.value)
    states = [dm.new_paged_state(cfg, 3, 12, 8) for _ in range(2)]
    rng = np.random.default_rng(13)
    prompt = rng.integers(0, cfg.vocab, (3, 6)).astype(np.int32)
    for state, d in zip(states, (dec, plain)):
        d.extend(prompt, state)
        d.extend(prompt[:1, :3], state, rows=range(1, 2))
    for step in range(6):
        if step == 4:
            for state in states:
                state.release(2)
        ids = rng.integers(0, cfg.vocab, (3, 1)).astype(np.int32)
        got = dec.extend(ids, states[0], graph=True)
        _lib.call("mfb_stream_sync", ctypes.c_void_p(stream.value))
        assert np.array_equal(got.numpy(), plain.extend(ids, states[1]).numpy()), step
    assert states[0].lengths == [12, 15, 2]
    with pytest.raises(ValueError, match="single tokens"):
        dec.extend(prompt, states[0], graph=True)
    with pytest.raises(ValueError, match="created stream|stream="):
        plain.extend(prompt[:, :1], states[1], graph=True)


@pytest.mark.parametrize("path", ["extend", "decode_one", "graph"])
def test_controls_apply_to_the_steps_logits(model, path):
    """Against the float64 controls of the same step's uncontrolled logits (the step is deterministic)."""
    import ctypes
    from minifield_training_b200 import _lib
    from oracle import paged as ref
    dm, cfg, params, dec = model
    stream = None
    if path == "graph":
        stream = ctypes.c_void_p()
        _lib.call("mfb_stream_create", ctypes.byref(stream))
        dec = dm.Decoder(cfg, params, stream=stream.value)
    rng = np.random.default_rng(11)
    prompt = rng.integers(0, cfg.vocab, (2, 8)).astype(np.int32)
    words = (cfg.vocab + 31) // 32
    controls = dict(history=np.concatenate([prompt, prompt[:, :3]], 1), prompt_len=np.array([8, 5], np.int32),
                    repetition=np.array([1.3, 0.8], np.float32), frequency=np.array([0.5, -0.25], np.float32),
                    presence=np.array([0.125, 1.0], np.float32), bias_ids=np.array([[4, -1], [7, 7]], np.int32),
                    bias_values=np.array([[2.0, 9.0], [1.0, -3.0]], np.float32),
                    mask=rng.integers(-2**31, 2**31, (1, words)).astype(np.int32),
                    mask_rows=np.array([0, -1], np.int32))
    got = []
    for c in (None, controls):
        if path == "extend":
            state = dm.new_paged_state(cfg, 2, 8, 8)
            dec.extend(prompt, state)
            out = dec.extend(prompt[:, :1], state, controls=c)
        else:
            state = dm.new_state(cfg, 2, 16)
            for t in range(2):
                out = dec.decode_one(prompt[:, t], state, controls=c if t else None, graph=path == "graph")
        _lib.call("mfb_stream_sync", ctypes.c_void_p(stream.value) if stream else None)
        got.append(out.numpy())
    want = ref.controlled_logits(got[0], **controls)
    kept = np.isfinite(want)
    assert np.array_equal(np.isneginf(got[1]), ~kept) and 0 < (~kept).sum() < want.size
    # A reciprocal (one step), its product and three sums: six half steps of values up to the terms' sum.
    size = np.abs(got[0]) * 1.3 + 3 * 0.5 + 1 + 3
    assert np.all(np.abs(got[1][kept] - want[kept]) <= (6 * 2.0**-24 * size)[kept])
