"""Fixed-capacity cached decoding of the LFM2.5 causal decoder on the B200 kernels.

Mirrors src/minifield_training/models/lfm2_5/decode.py: ``new_state`` (:75-134)
allocates zeroed per-layer caches (attention K/V [B, capacity, Hk, 64] bf16,
conv history [B, 2, C] bf16); ``Decoder.prefill`` (:373-416) runs a prompt of
T tokens per row through every block (:183-222), fills the caches and returns
the FP32 logits of the last prompt token; ``Decoder.decode_one`` (:419-466)
runs one token per row through every block (:225-262) and returns FP32 logits
of the tied head (model.py:818-829), advancing the state's valid length.

Prefill, per block over the B*T prompt tokens:

  conv       RMSNorm -> in_proj GEMM -> mfb_conv_causal (zero history in, the
             continuation history out) -> out_proj GEMM
  attention  RMSNorm -> fused q|k|v GEMM -> q/k RMSNorm + RoPE at 0..T-1 ->
             causal mfb_attn_fwd -> K/V rows copied into the cache
             (mfb_memcpy2d_d2d) -> out_proj GEMM

The reference pads the prompt to a power-of-two bucket (decode.py:63-67);
the padded tokens sit after every valid one and are masked, so causal
attention and the causal convolution never read them and the prompt runs
at its own length here. Decode, per block:

  conv       RMSNorm -> in_proj GEMM -> mfb_conv_step (gated causal conv over
             the history, history shifted in place) -> out_proj GEMM
  attention  RMSNorm -> fused q|k|v GEMM -> q/k RMSNorm + RoPE at the position
             -> mfb_decode_attn (cache append at the position, split-K
             attention over the valid length) -> out_proj GEMM
  then       residual + RMSNorm (one kernel) -> fused w1|w3 GEMM -> SwiGLU ->
             w2 GEMM, the residual folded into the next block's norm.

``Decoder.extend`` runs a chunk of one or more tokens per row over a
``PagedState``, whose rows keep their keys and values in pages of a pool shared
by all rows (and have lengths of their own): per attention block the q/k norm,
rotation and append are one pass (kernels.paged.paged_append) and the chunk
attends to the pages (paged_attention). A prompt is prefilled by one call or by
several chunks; one token per row is a decode step. The rotation's angles and
the norms are FP32, rounded once, so logits differ from the fixed-capacity
path's, which rounds step by step as the reference does, by bf16 roundings.

``controls`` of ``decode_one`` and ``extend`` (penalties, biases, grammar masks:
the keyword arguments of kernels.logits.process_logits) are applied in the pass
that widens the logits.

The masters are cast to bf16 once at construction (full_linear's cast,
kernels/linear.py:11); the q|k|v and w1|w3 products are single GEMMs over
concatenated rows.
"""

import ctypes
import weakref

import numpy as np

from .. import _lib
from ..device import DeviceArray
from ..kernels import logits as logit_controls
from ..kernels import paged
from .encoder import _fwd, rope_freqs

P = ctypes.c_void_p


class DecodeOverflow(ValueError):
    """A token would be written past the fixed cache capacity (decode.py:22-23)."""


def parameter_shapes(cfg) -> dict:
    """Reference decoder parameter names and shapes (models/lfm2_5/model.py:127-166)."""
    c, f, kv = cfg.hidden, cfg.ffn, cfg.kv_heads * cfg.head_dim
    shapes = {"model.embed_tokens.weight": (cfg.vocab, c), "model.embedding_norm.weight": (c,)}
    for i, kind in enumerate(cfg.layer_types):
        p = f"model.layers.{i}."
        shapes.update({p + "operator_norm.weight": (c,), p + "ffn_norm.weight": (c,),
                       p + "feed_forward.w1.weight": (f, c), p + "feed_forward.w3.weight": (f, c),
                       p + "feed_forward.w2.weight": (c, f)})
        if kind == "conv":
            shapes.update({p + "conv.in_proj.weight": (3 * c, c), p + "conv.out_proj.weight": (c, c),
                           p + "conv.conv.weight": (c, 1, cfg.conv_kernel)})
        else:
            shapes.update({p + "self_attn.q_proj.weight": (cfg.heads * cfg.head_dim, c),
                           p + "self_attn.k_proj.weight": (kv, c), p + "self_attn.v_proj.weight": (kv, c),
                           p + "self_attn.out_proj.weight": (c, cfg.heads * cfg.head_dim),
                           p + "self_attn.q_layernorm.weight": (cfg.head_dim,),
                           p + "self_attn.k_layernorm.weight": (cfg.head_dim,)})
    return shapes


def init_parameters(cfg, seed: int = 0) -> dict:
    """Random init: N(0, 0.02) for matrices, taps and the embedding table; ones for norm gains."""
    rng = np.random.default_rng(seed)
    out = {}
    for name, shape in parameter_shapes(cfg).items():
        if name.endswith("norm.weight") or name.endswith("layernorm.weight"):
            out[name] = np.ones(shape, np.float32)
        else:
            out[name] = rng.standard_normal(shape, dtype=np.float32) * np.float32(0.02)
    return out


class DecodeState:
    """Device caches of one prompt batch plus its logical position (decode.py:34-41).

    ``keys`` / ``values`` / ``history`` are per-layer lists (None where the
    layer has no such cache); ``valid_length`` is the number of written
    positions, which is also the position the next token takes.
    """

    def __init__(self, cfg, batch_size: int, capacity: int):
        if isinstance(capacity, bool) or not isinstance(capacity, int) or capacity <= 0 or capacity & (capacity - 1):
            raise ValueError("Cache capacity must be a positive power of two")
        if isinstance(batch_size, bool) or not isinstance(batch_size, int) or batch_size <= 0:
            raise ValueError("batch_size must be a positive integer")
        self.cfg, self.batch, self.capacity, self.valid_length = cfg, batch_size, capacity, 0
        self.keys, self.values, self.history = [], [], []
        for kind in cfg.layer_types:
            if kind == "full_attention":
                shape = (batch_size, capacity, cfg.kv_heads, cfg.head_dim)
                self.keys.append(DeviceArray.zeros(shape, "bfloat16"))
                self.values.append(DeviceArray.zeros(shape, "bfloat16"))
                self.history.append(None)
            else:
                self.keys.append(None)
                self.values.append(None)
                self.history.append(DeviceArray.zeros((batch_size, cfg.conv_kernel - 1, cfg.hidden), "bfloat16"))


def new_state(cfg, batch_size: int, capacity: int) -> DecodeState:
    """Zeroed fixed-capacity state (decode.py:75-134)."""
    return DecodeState(cfg, batch_size, capacity)


class PagedState:
    """Rows over a shared pool of pages (no counterpart in the reference).

    Every attention layer has a ``paged.PagedCache`` of ``num_pages`` pages of
    ``page_size`` tokens; a row takes pages as it grows, the same ones in every
    layer, up to ``max_pages`` (default: what the pool and the model's positions
    allow), and gives them back on ``release``. ``lengths`` holds each row's
    tokens; ``table`` its pages (-1 behind them), of which ``device_table`` is a
    copy that ``upload`` keeps up by the pages taken since, so that a step costs
    no more for a wide table; ``history`` the conv layers' two preceding inputs
    per row.
    """

    def __init__(self, cfg, batch_size: int, num_pages: int, page_size: int = 64, max_pages: int | None = None):
        for name, n in (("batch_size", batch_size), ("num_pages", num_pages), ("page_size", page_size),
                        ("max_pages", 1 if max_pages is None else max_pages)):
            if isinstance(n, bool) or not isinstance(n, int) or n <= 0:
                raise ValueError(f"{name} must be a positive integer")
        if batch_size > 8192:
            raise ValueError(f"batch_size {batch_size} above the supported 8192 rows")
        if page_size < 8 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two of at least 8")
        self.cfg, self.batch, self.page_size, self.num_pages = cfg, batch_size, page_size, num_pages
        self.max_pages = min(max_pages or num_pages, num_pages, self.pages(cfg.max_position_embeddings))
        self.lengths = [0] * batch_size
        self.table = np.full((batch_size, self.max_pages), -1, np.int32)
        self.device_table = DeviceArray.from_numpy(self.table)
        self._taken = []  # (row, first, count) of pages that device_table lacks
        self._free = list(range(num_pages - 1, -1, -1))
        self.caches, self.history = [], []
        for kind in cfg.layer_types:
            if kind == "full_attention":
                self.caches.append(paged.PagedCache.zeros(num_pages, page_size, cfg.kv_heads, cfg.head_dim))
                self.history.append(None)
            else:
                self.caches.append(None)
                self.history.append(DeviceArray.zeros((batch_size, cfg.conv_kernel - 1, cfg.hidden), "bfloat16"))
        _lib.call("mfb_stream_sync", None)  # any stream may use the pool from here on

    def pages(self, tokens: int) -> int:
        """Pages that hold ``tokens`` tokens of a row."""
        return -(-tokens // self.page_size)

    def grow(self, rows, tokens: int) -> None:
        """Takes the pages for ``tokens`` more tokens of each of ``rows``, or none at all (DecodeOverflow)."""
        rows, need = list(rows), []
        if tokens <= 0 or len(set(rows)) != len(rows) or any(not 0 <= row < self.batch for row in rows):
            raise ValueError(f"pages go to distinct rows of the batch of {self.batch}, for a positive number of tokens")
        for row in rows:
            total = self.lengths[row] + tokens
            if total > self.cfg.max_position_embeddings:
                raise ValueError("Logical length exceeds model max_position_embeddings")
            if self.pages(total) > self.max_pages:
                raise DecodeOverflow(f"Row {row} needs {self.pages(total)} pages of {self.page_size} tokens; "
                                     f"it may take {self.max_pages}")
            need.append(self.pages(total) - self.pages(self.lengths[row]))
        if sum(need) > len(self._free):
            raise DecodeOverflow(f"{sum(need)} pages needed, {len(self._free)} of {self.num_pages} free")
        for row, count in zip(rows, need):
            held = self.pages(self.lengths[row])
            self.lengths[row] += tokens
            if count:
                self.table[row, held:held + count] = [self._free.pop() for _ in range(count)]
                self._taken.append((row, held, count))

    def upload(self, stream=None) -> None:
        """Brings ``device_table`` up to the pages taken, in the order of ``stream``."""
        for row, first, count in self._taken:
            entries = self.table[row, first:first + count]
            _lib.call("mfb_memcpy_h2d", P(self.device_table.ptr + (row * self.max_pages + first) * entries.itemsize),
                      entries.ctypes.data_as(P), entries.nbytes, stream)
        self._taken.clear()

    def release(self, row: int) -> None:
        """Empties ``row`` for a new sequence: its pages go back to the pool."""
        if isinstance(row, bool) or not isinstance(row, int) or not 0 <= row < self.batch:
            raise ValueError(f"row {row} outside the batch of {self.batch}")
        self._free.extend(int(p) for p in self.table[row, :self.pages(self.lengths[row])][::-1])
        self.table[row] = -1
        self.lengths[row] = 0


def new_paged_state(cfg, batch_size: int, num_pages: int, page_size: int = 64, max_pages: int | None = None):
    """An empty PagedState of ``batch_size`` rows over ``num_pages`` pages of ``page_size`` tokens."""
    return PagedState(cfg, batch_size, num_pages, page_size, max_pages)


class Decoder:
    """Device weights of the decoder and the single-token step over a DecodeState."""

    def __init__(self, cfg, parameters: dict, *, stream=None):
        if cfg.head_dim != 64 or cfg.conv_kernel != 3:
            raise ValueError("this build decodes head_dim 64 with a 3-tap convolution")
        shapes = parameter_shapes(cfg)
        if set(parameters) != set(shapes):
            raise ValueError("Decoder parameter tree mismatch")
        for name, shape in shapes.items():
            if tuple(np.shape(parameters[name])) != shape:
                raise ValueError(f"Decoder parameter shape mismatch: {name}")
        self.cfg, self.stream = cfg, stream
        f32 = lambda a: DeviceArray.from_numpy(np.ascontiguousarray(a, np.float32), "float32")  # noqa: E731

        def bf16(*names):  # rows of the named matrices, concatenated, cast to bf16 on the device
            host = np.ascontiguousarray(np.concatenate([np.asarray(parameters[n], np.float32) for n in names]))
            src = f32(host)
            out = DeviceArray(host.shape, "bfloat16")
            _lib.call("mfb_cast_f32_bf16", P(src.ptr), P(out.ptr), host.size, None)
            return out

        self.embed = f32(parameters["model.embed_tokens.weight"])
        self.head = bf16("model.embed_tokens.weight")
        self.final_norm = f32(parameters["model.embedding_norm.weight"])
        self.freqs = DeviceArray.from_numpy(rope_freqs(cfg.rope_theta, cfg.head_dim), "float32")
        self.layers = []
        for i, kind in enumerate(cfg.layer_types):
            p = f"model.layers.{i}."
            L = {"kind": kind, "op_norm": f32(parameters[p + "operator_norm.weight"]),
                 "ffn_norm": f32(parameters[p + "ffn_norm.weight"]),
                 "w13": bf16(p + "feed_forward.w1.weight", p + "feed_forward.w3.weight"),
                 "w2": bf16(p + "feed_forward.w2.weight")}
            if kind == "conv":
                L["w_in"] = bf16(p + "conv.in_proj.weight")
                L["w_out"] = bf16(p + "conv.out_proj.weight")
                L["taps"] = f32(np.asarray(parameters[p + "conv.conv.weight"], np.float32)[:, 0, :])
            else:
                L["w_in"] = bf16(p + "self_attn.q_proj.weight", p + "self_attn.k_proj.weight",
                                 p + "self_attn.v_proj.weight")
                L["w_out"] = bf16(p + "self_attn.out_proj.weight")
                L["qn"] = f32(parameters[p + "self_attn.q_layernorm.weight"])
                L["kn"] = f32(parameters[p + "self_attn.k_layernorm.weight"])
            self.layers.append(L)
        _lib.call("mfb_device_sync")
        self._scratch, self._graphs, self._prefill_scratch, self._extend_scratch = {}, {}, {}, {}
        self._dead_graphs = []  # keys of graphs whose paged state is gone

    def _buffers(self, batch: int, capacity: int):
        key = (batch, capacity)
        if key not in self._scratch:
            cfg, E = self.cfg, DeviceArray
            c, f, h, hk = cfg.hidden, cfg.ffn, cfg.heads, cfg.kv_heads
            nq = (h + 2 * hk) * cfg.head_dim
            ws = _lib.lib().mfb_decode_workspace_size(batch, capacity, h, cfg.head_dim)
            gemm_ws = max(int(_lib.lib().mfb_gemm_workspace_size(batch, n, k))
                          for n, k in ((3 * c, c), (c, c), (nq, c), (c, h * cfg.head_dim), (2 * f, c), (c, f),
                                       (cfg.vocab, c)))
            meta = E((3, batch), "int32")  # ids, positions, lengths: one upload per step
            self._scratch[key] = dict(
                meta=meta, ids=meta.view(0, (batch,)), pos=meta.view(batch, (batch,)),
                lens=meta.view(2 * batch, (batch,)),
                x=E((batch, c), "bfloat16"), xb=E((batch, c), "bfloat16"), hn=E((batch, c), "bfloat16"),
                proj=E((batch, max(3 * c, nq)), "bfloat16"), mixed=E((batch, c), "bfloat16"),
                r=E((batch, c), "bfloat16"), mid=E((batch, c), "bfloat16"), h2=E((batch, c), "bfloat16"),
                gu=E((batch, 2 * f), "bfloat16"), a=E((batch, f), "bfloat16"), y=E((batch, c), "bfloat16"),
                q=E((batch, h, 64), "bfloat16"), k=E((batch, hk, 64), "bfloat16"), v=E((batch, hk, 64), "bfloat16"),
                o=E((batch, h * 64), "bfloat16"), rq=E((batch, h), "float32"), rk=E((batch, hk), "float32"),
                rstd=E((batch,), "float32"), enc=E((batch, c), "bfloat16"),
                logits16=E((batch, cfg.vocab), "bfloat16"), logits=E((batch, cfg.vocab), "float32"),
                ws=E((max(ws, 16),), "uint8"), gemm_ws=E((max(gemm_ws, 16),), "uint8"))
        return self._scratch[key]

    def _proj(self, x, w, out, m, n, k, B):
        """out[m, n] = x[m, k] . w[n, k]^T (bf16). With the batch's few rows the library runs the product
        swapped (the weight rows on the tensor core's 128-row side) and splits K through the step's
        workspace only for a deep weight (w2).

        On a created stream it launches as a programmatic dependent: the
        weight tiles stream in while the previous kernel (norm, SwiGLU, conv
        step or attention) finishes.
        """
        _lib.call("mfb_gemm_bf16_ws", P(x.ptr), _lib.MAJOR_K, k, P(w.ptr), _lib.MAJOR_K, k, P(out.ptr), n,
                  _lib.DTYPE_BF16, m, n, k, ctypes.c_float(1.0), None, _lib.GEMM_PDL if self.stream else 0,
                  P(B["gemm_ws"].ptr),
                  B["gemm_ws"].nbytes, self.stream)

    def _rms(self, x, res, w, sum_out, y, rstd, m):
        _lib.call("mfb_rmsnorm_fwd", P(x.ptr), P(res.ptr) if res is not None else None, P(w.ptr), None,
                  P(sum_out.ptr) if sum_out is not None else None, P(y.ptr), P(rstd.ptr), m, self.cfg.hidden,
                  ctypes.c_float(self.cfg.norm_eps), self.stream)

    def prefill(self, input_ids, state: DecodeState):
        """FP32 logits [B, vocab] of the token after the prompt; fills the caches of a fresh state.

        ``input_ids`` [B, T] int32; raises the reference's ValueErrors
        (decode.py:382-396) before any kernel runs.
        """
        cfg, s = self.cfg, self.stream
        if state.cfg != cfg:
            raise ValueError("Decode state does not match the decoder config")
        if state.valid_length != 0:
            raise ValueError("Prefill requires a fresh state")
        ids = np.asarray(input_ids)
        if ids.ndim != 2:
            raise ValueError("Prefill input_ids must have shape [batch, tokens]")
        b, t = ids.shape
        if t > cfg.max_position_embeddings:
            raise ValueError("Logical length exceeds model max_position_embeddings")
        if b != state.batch:
            raise ValueError("Prompt batch does not match cache batch")
        if t <= 0 or t > state.capacity:
            raise ValueError("Prompt length must fit the cache capacity")
        ids = np.ascontiguousarray(ids, np.int32)
        c, f, h, hk, hd = cfg.hidden, cfg.ffn, cfg.heads, cfg.kv_heads, cfg.head_dim
        m, nq, E = b * t, (h + 2 * hk) * hd, DeviceArray
        # Scratch sized for the reference's power-of-two prompt bucket
        # (decode.py:63-67) and kept per (batch, bucket): at most log2(capacity)
        # buffer sets per batch size, whatever the prompt lengths. A prompt uses
        # the leading b*t rows ([b, t] arrays stay contiguous with row stride t).
        bucket = 1 << (t - 1).bit_length()
        B = self._prefill_scratch.get((b, bucket))
        if B is None:
            mb = b * bucket
            B = dict(ids=E((mb,), "int32"), pos=E((mb,), "int32"), mask=E((mb,), "int32"),
                     qid=E((mb,), "int32"), kid=E((mb,), "int32"),
                     x=E((mb, c), "bfloat16"), xb=E((mb, c), "bfloat16"), hn=E((mb, c), "bfloat16"),
                     proj=E((mb, max(3 * c, nq)), "bfloat16"), mixed=E((mb, c), "bfloat16"),
                     r=E((mb, c), "bfloat16"), mid=E((mb, c), "bfloat16"), h2=E((mb, c), "bfloat16"),
                     gu=E((mb, 2 * f), "bfloat16"), a=E((mb, f), "bfloat16"), y=E((mb, c), "bfloat16"),
                     q=E((mb, h, hd), "bfloat16"), k=E((mb, hk, hd), "bfloat16"), v=E((mb, hk, hd), "bfloat16"),
                     o=E((mb, h * hd), "bfloat16"), lse=E((mb * h,), "float32"), rq=E((mb, h), "float32"),
                     rk=E((mb, hk), "float32"), rstd=E((mb,), "float32"), enc=E((mb, c), "bfloat16"),
                     last=E((b, c), "bfloat16"), logits16=E((b, cfg.vocab), "bfloat16"), ws=E((16,), "uint8"))
            self._prefill_scratch[(b, bucket)] = B
        need = int(_lib.lib().mfb_attn_workspace_size(b, t, t, h, hk, hd))
        if B["ws"].nbytes < need:
            B["ws"] = E((need,), "uint8")
        ws = B["ws"]
        for name, host in (("ids", ids.reshape(-1)), ("pos", np.tile(np.arange(t, dtype=np.int32), b)),
                           ("mask", np.ones((b, t), np.int32))):
            host = np.ascontiguousarray(host)
            _lib.call("mfb_memcpy_h2d", P(B[name].ptr), host.ctypes.data_as(P), host.nbytes, s)
        causal, off, pol = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
        _lib.call("mfb_attn_ids", _lib.MASK_CAUSAL, P(B["mask"].ptr), None, None, P(B["qid"].ptr),
                  P(B["kid"].ptr), b, t, t, 0, ctypes.byref(causal), ctypes.byref(off), ctypes.byref(pol), s)
        _lib.call("mfb_embed_gather", P(self.embed.ptr), P(B["ids"].ptr), P(B["x"].ptr), m, c, cfg.vocab, s)
        row_kv = hk * hd * 2  # bytes of one token's K (or V) row
        x, prev_mid, prev_y = B["x"], None, None
        for i, L in enumerate(self.layers):
            if prev_mid is None:
                self._rms(x, None, L["op_norm"], None, B["hn"], B["rstd"], m)
            else:
                self._rms(prev_mid, prev_y, L["op_norm"], x, B["hn"], B["rstd"], m)
            if L["kind"] == "conv":
                _fwd(B["hn"], L["w_in"], B["proj"], m, 3 * c, c, s)
                _lib.call("mfb_conv_causal", P(B["proj"].ptr), P(L["taps"].ptr), None, P(state.history[i].ptr),
                          P(B["mixed"].ptr), b, t, c, s)
                _fwd(B["mixed"], L["w_out"], B["r"], m, c, c, s)
            else:
                _fwd(B["hn"], L["w_in"], B["proj"], m, nq, c, s)
                _lib.call("mfb_qknorm_rope_fwd", P(B["proj"].ptr), nq, P(L["qn"].ptr), P(L["kn"].ptr),
                          P(B["pos"].ptr), P(self.freqs.ptr), P(B["q"].ptr), P(B["k"].ptr), P(B["v"].ptr),
                          P(B["rq"].ptr), P(B["rk"].ptr), m, h, hk, ctypes.c_float(cfg.norm_eps), s)
                _lib.call("mfb_attn_fwd", P(B["q"].ptr), P(B["k"].ptr), P(B["v"].ptr), P(B["o"].ptr),
                          P(B["lse"].ptr), P(B["qid"].ptr), P(B["kid"].ptr), b, t, t, h, hk, hd, causal.value,
                          off.value, pol.value, ctypes.c_float(hd ** -0.5), P(ws.ptr), ws.nbytes, s)
                for cache, src in ((state.keys[i], B["k"]), (state.values[i], B["v"])):
                    _lib.call("mfb_memcpy2d_d2d", P(cache.ptr), state.capacity * row_kv, P(src.ptr), t * row_kv,
                              t * row_kv, b, s)
                _fwd(B["o"], L["w_out"], B["r"], m, c, h * hd, s)
            self._rms(x, B["r"], L["ffn_norm"], B["mid"], B["h2"], B["rstd"], m)
            _fwd(B["h2"], L["w13"], B["gu"], m, 2 * f, c, s)
            _lib.call("mfb_swiglu_fwd", P(B["gu"].ptr), P(B["a"].ptr), m, f, s)
            _fwd(B["a"], L["w2"], B["y"], m, c, f, s)
            prev_mid, prev_y = B["mid"], B["y"]
            x = B["xb"] if x is B["x"] else B["x"]
        self._rms(prev_mid, prev_y, self.final_norm, x, B["enc"], B["rstd"], m)
        _lib.call("mfb_memcpy2d_d2d", P(B["last"].ptr), c * 2, P(B["enc"].ptr + (t - 1) * c * 2), t * c * 2, c * 2,
                  b, s)  # the last prompt token of every row
        _fwd(B["last"], self.head, B["logits16"], b, cfg.vocab, c, s)
        logits = DeviceArray((b, cfg.vocab), "float32")
        _lib.call("mfb_cast_bf16_f32", P(B["logits16"].ptr), P(logits.ptr), b * cfg.vocab, s)
        state.valid_length = t
        return logits

    def extend(self, input_ids, state: PagedState, *, rows=None, controls=None, out=None, graph: bool = False):
        """FP32 logits [R, vocab] after the last of T new tokens per row; fills pages and advances the state.

        ``input_ids`` [R, T] int32 continue ``rows`` (a range of state rows, all
        by default), each at its own length: a prompt or a part of one, or one
        decoded token. DecodeOverflow when the pool or a row's table is full,
        like any other refusal, comes before anything runs and leaves the state
        as it was; what the attention clamps or gives up on while it runs is
        recorded for kernels.paged.paged_attention_status. ``controls``: keyword
        arguments of kernels.logits.process_logits for the returned logits. ``out`` (a
        float32 [R, vocab] DeviceArray) receives them. ``graph=True`` replays a
        single-token step (T = 1) as one CUDA graph, captured on the first call
        for these rows of this state (needs a created stream).
        """
        cfg, s = self.cfg, self.stream
        if state.cfg != cfg:
            raise ValueError("Decode state does not match the decoder config")
        rows = range(state.batch) if rows is None else rows
        if not isinstance(rows, range) or rows.step != 1 or not rows or rows.start < 0 or rows.stop > state.batch:
            raise ValueError(f"rows must be a non-empty range of step 1 within the {state.batch} rows of the state")
        ids = np.asarray(input_ids)
        if ids.ndim != 2 or ids.shape[0] != len(rows) or ids.shape[1] <= 0:
            raise ValueError("extend input_ids must have shape [rows, tokens] matching the rows of the state")
        b, t = ids.shape
        if out is not None and (not isinstance(out, DeviceArray) or out.shape != (b, cfg.vocab)
                                or out.dtype != "float32" or out.ptr % 16):
            raise ValueError("out must be a 16-byte aligned float32 [rows, vocab] device array")
        if graph and (not s or t != 1):
            raise ValueError("graph replay takes single tokens and needs Decoder(stream=...) from mfb_stream_create")
        controls = self._controls(controls, b)
        _lib.call("mfb_paged_attn_check", b * t, b, t, state.max_pages, state.num_pages, state.page_size, cfg.heads,
                  cfg.kv_heads, cfg.head_dim)
        fresh = []  # [first, count] of neighbouring rows that begin a sequence
        for row in rows:
            if state.lengths[row] == 0:
                if fresh and sum(fresh[-1]) == row:
                    fresh[-1][1] += 1
                else:
                    fresh.append([row, 1])
        B = self._extend_buffers(b, t, graph)
        logits = out if out is not None else DeviceArray((b, cfg.vocab), "float32")
        state.grow(rows, t)  # what can fail for lack of memory is behind us
        meta = np.concatenate([ids.reshape(-1).astype(np.int32), np.arange(b + 1, dtype=np.int32) * t,
                               np.asarray(state.lengths[rows.start:rows.stop], np.int32)])
        _lib.call("mfb_memcpy_h2d", P(B["meta"].ptr), meta.ctypes.data_as(P), meta.nbytes, s)
        state.upload(s)
        for history in state.history:
            if history is not None:
                nbytes = history.nbytes // state.batch
                for first, count in fresh:
                    _lib.call("mfb_memset", P(history.ptr + first * nbytes), 0, count * nbytes, s)
        if graph:
            key = ("paged", b, rows.start, state.max_pages, state.num_pages, state.page_size,
                   state.device_table.ptr) + tuple(
                h.ptr if c is None else (c.keys.ptr, c.values.ptr) for c, h in zip(state.caches, state.history))
            if self._dead_graphs:
                _lib.call("mfb_stream_sync", P(s))  # their last replays may still run
                while self._dead_graphs:
                    _lib.call("mfb_graph_destroy", P(self._graphs.pop(self._dead_graphs.pop())))
            g = self._graphs.get(key)
            if g is None:
                _lib.call("mfb_graph_begin", P(s))
                try:
                    self._extend_layers(B, state, rows, t)
                finally:
                    g_ = P()
                    _lib.call("mfb_graph_end", P(s), ctypes.byref(g_))
                g = self._graphs[key] = g_.value
                weakref.finalize(state, self._dead_graphs.append, key).atexit = False
            _lib.call("mfb_graph_launch", P(g), P(s))
        else:
            self._extend_layers(B, state, rows, t)
        return self._widen(B["logits16"].view(0, (b, cfg.vocab)), logits, controls)

    def _extend_layers(self, B, state: PagedState, rows, t: int):
        """Every layer over the ``t`` uploaded tokens of ``rows``; bf16 logits of the last ones in B["logits16"]."""
        cfg, s, b = self.cfg, self.stream, len(rows)
        c, f, h, hk, hd = cfg.hidden, cfg.ffn, cfg.heads, cfg.kv_heads, cfg.head_dim
        m, nq = b * t, (h + 2 * hk) * hd
        ids_d, cu = B["meta"].view(0, (m,)), B["meta"].view(m, (b + 1,))
        lens = B["meta"].view(m + b + 1, (b,))
        table = state.device_table.view(rows.start * state.max_pages, (b, state.max_pages))

        def proj(x, w, y, n, k):
            if m <= 64:
                self._proj(x, w, y, m, n, k, B)
            else:
                _fwd(x, w, y, m, n, k, s)

        x, spare, prev_mid, prev_y = B["x"], B["xb"], None, None
        _lib.call("mfb_embed_gather", P(self.embed.ptr), P(ids_d.ptr), P(x.ptr), m, c, cfg.vocab, s)
        for i, L in enumerate(self.layers):
            if prev_mid is None:
                self._rms(x, None, L["op_norm"], None, B["hn"], B["rstd"], m)
            else:
                self._rms(prev_mid, prev_y, L["op_norm"], x, B["hn"], B["rstd"], m)
            if L["kind"] == "conv":
                proj(B["hn"], L["w_in"], B["proj"], 3 * c, c)
                nbytes = state.history[i].nbytes // state.batch
                history = state.history[i].ptr + rows.start * nbytes
                if t == 1:
                    _lib.call("mfb_conv_step", P(B["proj"].ptr), P(L["taps"].ptr), P(history), P(B["mixed"].ptr),
                              b, c, s)
                else:  # the tail it leaves must not alias the history it starts from
                    _lib.call("mfb_conv_causal", P(B["proj"].ptr), P(L["taps"].ptr), P(history), P(B["tail"].ptr),
                              P(B["mixed"].ptr), b, t, c, s)
                    _lib.call("mfb_memcpy_d2d", P(history), P(B["tail"].ptr), b * nbytes, s)
                proj(B["mixed"], L["w_out"], B["r"], c, c)
            else:
                proj(B["hn"], L["w_in"], B["proj"], nq, c)
                qkv, q, o = B["proj"].view(0, (m, nq)), B["q"].view(0, (m, h, hd)), B["o"].view(0, (m, h, hd))
                paged.paged_append(qkv, state.caches[i], cu, lens, table, heads=h, freqs=self.freqs,
                                   q_weight=L["qn"], k_weight=L["kn"], eps=cfg.norm_eps, out=q, stream=s)
                paged.paged_attention(q, state.caches[i], cu, lens, table, max_q=t, out=o, workspace=B["ws"],
                                      stream=s)
                proj(B["o"], L["w_out"], B["r"], c, h * hd)
            self._rms(x, B["r"], L["ffn_norm"], B["mid"], B["h2"], B["rstd"], m)
            proj(B["h2"], L["w13"], B["gu"], 2 * f, c)
            _lib.call("mfb_swiglu_fwd", P(B["gu"].ptr), P(B["a"].ptr), m, f, s)
            proj(B["a"], L["w2"], B["y"], c, f)
            prev_mid, prev_y = B["mid"], B["y"]
            x, spare = spare, x
        self._rms(prev_mid, prev_y, self.final_norm, x, B["enc"], B["rstd"], m)
        # Logits of the last token of every row.
        _lib.call("mfb_memcpy2d_d2d", P(B["last"].ptr), c * 2, P(B["enc"].ptr + (t - 1) * c * 2), t * c * 2, c * 2,
                  b, s)
        if b <= 64:
            self._proj(B["last"], self.head, B["logits16"], b, cfg.vocab, c, B)
        else:
            _fwd(B["last"], self.head, B["logits16"], b, cfg.vocab, c, s)

    def _extend_buffers(self, b: int, t: int, graph: bool = False):
        """Scratch of ``extend`` for b x t tokens.

        Calls are serial on the decoder's stream, so one set serves them all and
        grows to the largest, in steps of an eighth at most. A captured step needs
        buffers that stay: a set of its own per power of two of rows.
        """
        cfg, E = self.cfg, DeviceArray
        c, f, h, hk, hd = cfg.hidden, cfg.ffn, cfg.heads, cfg.kv_heads, cfg.head_dim
        nq = (h + 2 * hk) * hd

        def rounded(x):
            step = max((1 << (x - 1).bit_length()) >> 4, 1)
            return -(-x // step) * step

        r, n = (rounded(b), rounded(b * t)) if not graph else (1 << (b - 1).bit_length(),) * 2
        key = r if graph else None
        B = self._extend_scratch.get(key)
        if B is None or B["rows"] < r or B["tokens"] < n:
            if B is not None:
                r, n = max(r, B["rows"]), max(n, B["tokens"])
                B = None
                del self._extend_scratch[key]  # before the larger one is allocated

            def bf(cols, rows=n):
                return E((rows, cols), "bfloat16")

            size = _lib.lib().mfb_gemm_workspace_size
            gemm = [int(size(min(n, 64), w, k)) for w, k in (
                (3 * c, c), (c, c), (nq, c), (c, h * hd), (2 * f, c), (c, f))]
            gemm.append(int(size(min(r, 64), cfg.vocab, c)))
            B = self._extend_scratch[key] = dict(
                rows=r, tokens=n, meta=E((n + 2 * r + 1,), "int32"), x=bf(c), xb=bf(c), hn=bf(c),
                proj=E((n * max(3 * c, nq),), "bfloat16"), mixed=bf(c), tail=bf((cfg.conv_kernel - 1) * c, r),
                r=bf(c), mid=bf(c), h2=bf(c), gu=bf(2 * f), a=bf(f), y=bf(c), q=bf(h * hd), o=bf(h * hd),
                rstd=E((n,), "float32"), enc=bf(c), last=bf(c, r), logits16=bf(cfg.vocab, r),
                gemm_ws=E((max(*gemm, 16),), "uint8"), ws=E((16,), "uint8"))
        need = paged.paged_attention_workspace_size(n if graph else b * t, r if graph else b, t, h, hk, hd)
        if B["ws"].nbytes < need:
            B["ws"] = E((need,), "uint8")
        return B

    def _controls(self, controls, rows: int):
        """Checked controls, before the state changes."""
        if not controls:
            return None
        return logit_controls.prepare_controls(rows, self.cfg.vocab, stream=self.stream, **controls)

    def _widen(self, logits16, logits, controls):
        """FP32 ``logits`` of the bf16 ones, under ``controls`` when given."""
        if controls is not None:
            return logit_controls.process_logits(logits16, out=logits, stream=self.stream, controls=controls)
        _lib.call("mfb_cast_bf16_f32", P(logits16.ptr), P(logits.ptr), logits.size, self.stream)
        return logits

    def decode_one(self, input_ids, state: DecodeState, *, out=None, graph: bool = False, controls=None):
        """FP32 logits [B, vocab] of the next token for each row; writes the caches and advances the state.

        ``out`` (a float32 [B, vocab] DeviceArray) receives the logits instead
        of a new array. ``graph=True`` replays the step as one CUDA graph,
        captured on the first call for this state's caches (needs a created
        stream); the step reads its token ids, positions and lengths from
        device buffers uploaded before each replay, so one graph serves every
        step (and one every step with controls, which apply behind the replay).
        ``controls``: keyword arguments of kernels.logits.process_logits for the
        returned logits.
        """
        cfg, s = self.cfg, self.stream
        if state.cfg != cfg:
            raise ValueError("Decode state does not match the decoder config")
        if state.valid_length >= cfg.max_position_embeddings:
            raise ValueError("Decode position exceeds model max_position_embeddings")
        if state.valid_length >= state.capacity:
            raise DecodeOverflow(f"Cannot decode at position {state.valid_length}; capacity is {state.capacity}")
        ids = np.asarray(input_ids, np.int32)
        if ids.ndim == 2 and ids.shape[1] == 1:
            ids = ids[:, 0]
        if ids.ndim != 1 or ids.shape[0] != state.batch:
            raise ValueError("decode_one input_ids must have shape [batch] or [batch, 1] matching the state")
        b = state.batch
        if out is not None and (tuple(out.shape) != (b, cfg.vocab) or out.dtype != "float32"):
            raise ValueError("out must be a float32 [batch, vocab] device array")
        if graph and not s:
            raise ValueError("graph replay needs Decoder(stream=...) from mfb_stream_create")
        controls = self._controls(controls, b)
        B = self._buffers(b, state.capacity)
        pos = state.valid_length
        meta = np.ascontiguousarray(np.stack([ids, np.full(b, pos, np.int32), np.full(b, pos + 1, np.int32)]))
        _lib.call("mfb_memcpy_h2d", P(B["meta"].ptr), meta.ctypes.data_as(P), meta.nbytes, s)
        logits = out if out is not None else DeviceArray((b, cfg.vocab), "float32")
        if graph:
            key = (b, state.capacity, controls is None) + tuple(a.ptr for a in (*state.keys, *state.values, *state.history)
                                                                if a is not None)
            g = self._graphs.get(key)
            if g is None:
                _lib.call("mfb_graph_begin", P(s))
                try:
                    self._step(B, state, B["logits"] if controls is None else None)
                finally:
                    g_ = P()
                    _lib.call("mfb_graph_end", P(s), ctypes.byref(g_))
                g = self._graphs[key] = g_.value
            _lib.call("mfb_graph_launch", P(g), P(s))
            if controls is None:
                _lib.call("mfb_memcpy_d2d", P(logits.ptr), P(B["logits"].ptr), logits.nbytes, s)
        else:
            self._step(B, state, logits if controls is None else None)
        if controls is not None:
            self._widen(B["logits16"], logits, controls)
        state.valid_length = pos + 1
        return logits

    def _step(self, B, state: DecodeState, logits):
        """The device work of one decode step (token ids, positions, lengths already in B)."""
        cfg, s = self.cfg, self.stream
        b, c, f, h, hk = state.batch, cfg.hidden, cfg.ffn, cfg.heads, cfg.kv_heads
        nq = (h + 2 * hk) * cfg.head_dim
        _lib.call("mfb_embed_gather", P(self.embed.ptr), P(B["ids"].ptr), P(B["x"].ptr), b, c, cfg.vocab, s)
        x, prev_mid, prev_y = B["x"], None, None
        for i, L in enumerate(self.layers):
            # Block input (the previous block's mid + FFN output) and its operator norm.
            if prev_mid is None:
                self._rms(x, None, L["op_norm"], None, B["hn"], B["rstd"], b)
            else:
                self._rms(prev_mid, prev_y, L["op_norm"], x, B["hn"], B["rstd"], b)
            if L["kind"] == "conv":
                self._proj(B["hn"], L["w_in"], B["proj"], b, 3 * c, c, B)
                _lib.call("mfb_conv_step", P(B["proj"].ptr), P(L["taps"].ptr), P(state.history[i].ptr),
                          P(B["mixed"].ptr), b, c, s)
                self._proj(B["mixed"], L["w_out"], B["r"], b, c, c, B)
            else:
                self._proj(B["hn"], L["w_in"], B["proj"], b, nq, c, B)
                _lib.call("mfb_qknorm_rope_fwd", P(B["proj"].ptr), nq, P(L["qn"].ptr), P(L["kn"].ptr),
                          P(B["pos"].ptr), P(self.freqs.ptr), P(B["q"].ptr), P(B["k"].ptr), P(B["v"].ptr),
                          P(B["rq"].ptr), P(B["rk"].ptr), b, h, hk, ctypes.c_float(cfg.norm_eps), s)
                _lib.call("mfb_decode_attn", P(B["q"].ptr), P(state.keys[i].ptr), P(state.values[i].ptr),
                          P(B["k"].ptr), P(B["v"].ptr), P(B["pos"].ptr), P(B["lens"].ptr), P(B["o"].ptr), b,
                          state.capacity, h, hk, cfg.head_dim, ctypes.c_float(cfg.head_dim ** -0.5),
                          P(B["ws"].ptr), B["ws"].nbytes, s)
                self._proj(B["o"], L["w_out"], B["r"], b, c, h * cfg.head_dim, B)
            self._rms(x, B["r"], L["ffn_norm"], B["mid"], B["h2"], B["rstd"], b)
            self._proj(B["h2"], L["w13"], B["gu"], b, 2 * f, c, B)
            _lib.call("mfb_swiglu_fwd", P(B["gu"].ptr), P(B["a"].ptr), b, f, s)
            self._proj(B["a"], L["w2"], B["y"], b, c, f, B)
            prev_mid, prev_y = B["mid"], B["y"]
            x = B["xb"] if x is B["x"] else B["x"]  # the next block's input buffer (ping-pong)
        self._rms(prev_mid, prev_y, self.final_norm, x, B["enc"], B["rstd"], b)
        self._proj(B["enc"], self.head, B["logits16"], b, cfg.vocab, c, B)
        if logits is not None:
            _lib.call("mfb_cast_bf16_f32", P(B["logits16"].ptr), P(logits.ptr), b * cfg.vocab, s)

    def close(self):
        """Release the captured decode graphs and the scratch of ``extend``."""
        graphs, self._graphs, self._dead_graphs = getattr(self, "_graphs", {}), {}, []
        for g in graphs.values():
            if _lib._lib is not None:
                _lib.lib().mfb_graph_destroy(P(g))
        self._extend_scratch = {}

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def prefill(decoder: Decoder, input_ids, state: DecodeState):
    """``(logits, state)`` like models/lfm2_5/decode.py:373 (the state's device caches are filled in place)."""
    return decoder.prefill(input_ids, state), state


def decode_one(decoder: Decoder, input_ids, state: DecodeState):
    """``(logits, state)`` like models/lfm2_5/decode.py:419 (the state's device caches are updated in place)."""
    return decoder.decode_one(input_ids, state), state


def extend(decoder: Decoder, input_ids, state: PagedState, *, rows=None, controls=None):
    """``(logits, state)`` of ``Decoder.extend``."""
    return decoder.extend(input_ids, state, rows=rows, controls=controls), state


__all__ = ["DecodeOverflow", "DecodeState", "Decoder", "PagedState", "decode_one", "extend", "init_parameters",
           "new_paged_state", "new_state", "prefill", "parameter_shapes"]
