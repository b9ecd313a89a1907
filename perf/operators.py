"""Workloads of the rotary, paged-cache and logit operators: listed and drawn cases, inputs, plain forms and exact values.

``run`` computes a case in elementary torch operations where ``own`` is false,
and through ``minifield_training_b200.kernels`` where it is true.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": (torch.bfloat16, "bfloat16"), "fp16": (torch.float16, "float16"), "fp32": (torch.float32, "float32")}
EPS = 1e-5


def listed():
    return [
        # Training: the whole q|k|v projection of a layer, forward and backward. The small one is a
        # short fine-tuning row; the ordinary one the 8 x 2048 packed tokens of the encoder's shapes;
        # the third a long-context variant (half the head rotated, interleaved, positions past 2^20).
        {"name": "rotary train 37", "op": "rotary", "tokens": 37, "heads": 16, "kv_heads": 8, "head_dim": 64,
         "part": 1.0, "interleaved": False, "norm": True, "far": 0, "factor": 1.0, "dtype": "bf16"},
        {"name": "rotary train 16384", "op": "rotary", "tokens": 16384, "heads": 16, "kv_heads": 8, "head_dim": 64,
         "part": 1.0, "interleaved": False, "norm": True, "far": 0, "factor": 1.0, "dtype": "bf16"},
        {"name": "rotary train far 5001", "op": "rotary", "tokens": 5001, "heads": 12, "kv_heads": 4, "head_dim": 128,
         "part": 0.5, "interleaved": True, "norm": False, "far": 1 << 20, "factor": 8.0, "dtype": "fp16"},
        # One decode step of 64 rows, and a ragged chunked prefill: keys and values into the pages.
        {"name": "append step 64", "op": "append", "batch": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 256, "kv_hi": 4096,
         "lengths": 1, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 16, "head_major": False, "part": 1.0,
         "interleaved": False, "norm": True, "dtype": "bf16", "pad": 0},
        {"name": "append chunks", "op": "append", "batch": 7, "q_lo": 700, "q_hi": 2048, "kv_lo": 2100, "kv_hi": 9000,
         "lengths": 2, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 64, "head_major": True, "part": 1.0,
         "interleaved": False, "norm": True, "dtype": "bf16", "pad": 5},
        # Attention over pages: one user's next token after a short prompt (latency); the 64-row decode
        # step; a mixed batch of chunks in fp16 with wide heads; a chunk far into a long document; and
        # the prefill chunks of two long prompts (the largest).
        {"name": "attention step 1", "op": "attention", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 200, "kv_hi": 200,
         "lengths": 3, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 16, "head_major": False, "dtype": "bf16",
         "pad": 0},
        {"name": "attention step 64", "op": "attention", "batch": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 256,
         "kv_hi": 4096, "lengths": 1, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 16, "head_major": False,
         "dtype": "bf16", "pad": 0},
        {"name": "attention mixed fp16", "op": "attention", "batch": 9, "q_lo": 1, "q_hi": 300, "kv_lo": 301,
         "kv_hi": 5000, "lengths": 4, "heads": 16, "kv_heads": 4, "head_dim": 128, "page": 32, "head_major": True,
         "dtype": "fp16", "pad": 3},
        {"name": "attention far chunk", "op": "attention", "batch": 1, "q_lo": 250, "q_hi": 250, "kv_lo": 60001,
         "kv_hi": 60001, "lengths": 5, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 64, "head_major": False,
         "dtype": "bf16", "pad": 0},
        {"name": "attention prefill", "op": "attention", "batch": 2, "q_lo": 2048, "q_hi": 2048, "kv_lo": 8192,
         "kv_hi": 8192, "lengths": 6, "heads": 16, "kv_heads": 8, "head_dim": 64, "page": 64, "head_major": False,
         "dtype": "bf16", "pad": 0},
        # Logits before sampling: one user's token, and a 64-row step with long histories and grammars.
        {"name": "logits 1", "op": "logits", "rows": 1, "vocab": 65536, "history": 300, "bias": 8, "grammar": True,
         "dtype": "bf16"},
        {"name": "logits 64", "op": "logits", "rows": 64, "vocab": 65536, "history": 4096, "bias": 100,
         "grammar": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "logits"])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (16, 4), (12, 4), (8, 8), (10, 2), (14, 2), (8, 1)])
    head_dim = rng.choice([64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    turn = {"part": rng.choice([1.0, 1.0, 0.5, 0.25]), "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.6}
    if op == "rotary":
        return {"op": op, "tokens": _log(rng, 1, 9000 * 64 // head_dim), "heads": heads, "kv_heads": kv_heads,
                "head_dim": head_dim, **turn, "far": rng.choice([0, 0, 1 << 17, 1 << 20]),
                "factor": rng.choice([1.0, 4.0, 32.0]), "dtype": dtype}
    if op == "logits":
        vocab = rng.choice([65536, 65536, 32003, 50257, 128256])
        return {"op": op, "rows": _log(rng, 1, 64 * 65536 // max(vocab, 65536)), "vocab": vocab,
                "history": _log(rng, 1, 4096), "bias": rng.choice([0, 1, 17, 100]), "grammar": rng.random() < 0.6,
                "dtype": rng.choice(["bf16", "fp32", "fp16"])}
    paged = {"lengths": rng.randrange(1 << 20), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
             "page": rng.choice([8, 16, 32, 64, 128]), "head_major": rng.random() < 0.4, "dtype": dtype,
             "pad": rng.choice([0, 0, 3])}
    if op == "append":
        batch = _log(rng, 1, 64)
        q_hi = _log(rng, 1, max(1, 9000 // batch))
        return {"op": op, "batch": batch, "q_lo": rng.choice([0, 1]), "q_hi": q_hi, "kv_lo": q_hi,
                "kv_hi": q_hi + _log(rng, 1, 2000), **turn, **paged}
    while True:
        batch, q_hi, kv_hi = _log(rng, 1, 64), _log(rng, 1, 2048), _log(rng, 1, 60000)
        q_hi = 1 if rng.random() < 0.35 else q_hi
        kv_lo = max(1, kv_hi // rng.choice([1, 2, 20]))
        # Score entries of the padded plain form, and cache rows, of the largest listed case at most.
        if q_hi <= kv_lo and batch * q_hi * kv_hi <= 33_000_000 and batch * kv_hi <= 260_000:
            return {"op": op, "batch": batch, "q_lo": rng.choice([0, 1, q_hi]), "q_hi": q_hi, "kv_lo": kv_lo,
                    "kv_hi": kv_hi, **paged}


def _lengths(case):
    """Per-sequence counts of new tokens and of all tokens, from the case alone."""
    rng = random.Random(case["lengths"])
    q = [case["q_lo"] if case["q_lo"] == case["q_hi"] else min(case["q_hi"], max(case["q_lo"], _log(
        rng, max(1, case["q_lo"]), case["q_hi"]) - (1 if case["q_lo"] == 0 and rng.random() < 0.2 else 0)))
        for _ in range(case["batch"])]
    kv = [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(case["batch"])]
    if not any(q):
        q[0] = 1
    return q, kv


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        read = n * size + (n / 8 if case["grammar"] else 0) + case["rows"] * 4 * (case["history"] + 2 * case["bias"])
        return {"bytes": read + 4 * n, "flops": 4 * n}
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * (h + 2 * hk) * d
        return {"bytes": 5 * n * size + 4 * case["tokens"], "flops": 24 * n}
    q, kv = _lengths(case)
    tables = 8 * case["batch"] + 4 * sum(-(-s // case["page"]) for s in kv)
    if case["op"] == "append":
        n = sum(q) * (h + 2 * hk) * d
        return {"bytes": 2 * n * size + tables, "flops": 10 * n}
    pairs = sum(a * s - a * (a - 1) // 2 for a, s in zip(q, kv))
    live = sum(s for a, s in zip(q, kv) if a)
    return {"bytes": 2 * sum(q) * h * d * size + 2 * live * hk * d * size + tables, "flops": 4 * h * d * pairs}


def _frequencies(rotary_dim, factor):
    """theta ** (-2i / R), the long waves interpolated by ``factor`` (float32)."""
    base = 1e6 ** (-np.arange(0, rotary_dim, 2, dtype=np.float64) / rotary_dim)
    if factor > 1.0:
        turns = 8192 * base / (2 * math.pi)  # over the original context
        keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
        base = base * (keep + (1.0 - keep) / factor)
    return base.astype(np.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dt, name = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = {"case": dict(case), "name": name}
    if case["op"] == "logits":
        b, v, n = case["rows"], case["vocab"], case["history"]
        s["logits"] = (normal(b, v, dtype=torch.float32) * 3.0).to(dt)
        # Zipf-like token ids, so that histories repeat themselves.
        u = torch.rand(b, n, generator=g, device="cuda", dtype=torch.float64)
        s["history"] = (torch.exp(u * math.log(v)) - 1.0).long().clamp(0, v - 1).int()
        used = [rng.randint(0, n) if b > 1 else n for _ in range(b)]
        s["history_len"] = ints(used)
        s["prompt_len"] = ints([rng.randint(0, u) for u in used])
        s["repetition"] = 1.0 + torch.rand(b, generator=g, device="cuda") * 0.3
        s["frequency"] = torch.rand(b, generator=g, device="cuda") * 0.5
        s["presence"] = torch.rand(b, generator=g, device="cuda") * 0.5
        if case["bias"]:
            ids = torch.rand(b, v, generator=g, device="cuda").topk(case["bias"], dim=1).indices.int()
            s["bias_ids"], s["bias_values"] = ids.contiguous(), normal(b, case["bias"], dtype=torch.float32) * 5.0
        if case["grammar"]:
            s["mask"] = torch.randint(-(1 << 31), 1 << 31, (b, (v + 31) // 32), generator=g, device="cuda").int()
        s["out"] = torch.empty(b, v, dtype=torch.float32, device="cuda")
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] in ("rotary", "append"):
        s["rotary_dim"] = int(d * case["part"])
        f = _frequencies(s["rotary_dim"], case.get("factor", 1.0))
        s["freqs"] = torch.from_numpy(f).cuda()
        s["amplitude"] = 1.0 + 0.1 * math.log(case["factor"]) if case.get("factor", 1.0) > 1.0 else 1.0
        if case["norm"]:
            s["wq"], s["wk"] = (1.0 + 0.2 * normal(d, dtype=torch.float32) for _ in range(2))
    if case["op"] == "rotary":
        m = case["tokens"]
        s["qkv"] = normal(m, (h + 2 * hk) * d)
        start = rng.randint(0, case["far"]) if case["far"] else 0
        s["positions"] = (torch.arange(m, device="cuda") % max(1, min(m, 2048)) + start).int()
        s["dq"], s["dk"], s["dv"] = normal(m, h, d), normal(m, hk, d), normal(m, hk, d)
        s["outs"] = [torch.empty_like(s[k]) for k in ("dq", "dk", "dv", "qkv")]
        s["dw"] = [torch.empty(d, dtype=torch.float32, device="cuda") for _ in range(2)]
        return s
    q, kv = _lengths(case)
    n = sum(q) + case["pad"]
    page, b = case["page"], case["batch"]
    need = [-(-x // page) for x in kv]
    total = sum(need) + 3
    order = list(range(total))
    rng.shuffle(order)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    s["table"], s["seq_lens"] = table.cuda(), ints(kv)
    s["cu_q"] = ints([sum(q[:i]) for i in range(b + 1)])
    s["max_q"] = case["q_hi"]
    shape = (total, hk, page, d) if case["head_major"] else (total, page, hk, d)
    s["keys"], s["values"] = normal(*shape), normal(*shape)
    if case["op"] == "append":
        s["qkv"] = normal(n, (h + 2 * hk) * d)
    else:
        s["q"] = normal(n, h, d)
    s["out"] = torch.zeros(n, h, d, dtype=dt, device="cuda")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------


def _turn(s, positions, inverse=False):
    """cos, sin of position x frequency: the angle in 64 bits, the rest in 32."""
    angle = positions.double()[:, None] * s["freqs"].double()[None, :]
    c, n = angle.cos().float() * s["amplitude"], angle.sin().float() * s["amplitude"]
    return c[:, None, :], -n[:, None, :] if inverse else n[:, None, :]


def _rotate(s, x, cs):
    r, (c, n) = s["rotary_dim"], cs
    a, rest = x[..., :r], x[..., r:]
    if s["case"]["interleaved"]:
        x1, x2 = a[..., 0::2], a[..., 1::2]
        y = torch.stack([x1 * c - x2 * n, x2 * c + x1 * n], dim=-1).flatten(-2)
    else:
        x1, x2 = a[..., : r // 2], a[..., r // 2:]
        y = torch.cat([x1 * c - x2 * n, x2 * c + x1 * n], dim=-1)
    return torch.cat([y, rest], dim=-1)


def _heads(s, x):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    x = x.view(x.shape[0], h + 2 * hk, d)
    return x[:, :h], x[:, h:h + hk], x[:, h + hk:]


def _normed(x, w):
    """(x^, r) with x^ = x r, r = 1 / sqrt(mean x^2 + eps); without gains x itself."""
    if w is None:
        return x, None
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * r, r


def _plain_rotary(s):
    dt = s["qkv"].dtype
    cs, back = _turn(s, s["positions"]), _turn(s, s["positions"], inverse=True)
    q, k, v = _heads(s, s["qkv"])

    def one(x, dy, w):
        n, r = _normed(x.float(), w)
        y = _rotate(s, n if w is None else n * w, cs)
        dn = _rotate(s, dy.float(), back)
        if w is None:
            return y, dn, None
        dnw = dn * w
        dx = r * (dnw - n * (dnw * n).mean(-1, keepdim=True))
        return y, dx, (dn * n).double().sum((0, 1)).float()

    yq, dxq, dwq = one(q, s["dq"], s.get("wq"))
    yk, dxk, dwk = one(k, s["dk"], s.get("wk"))
    dqkv = torch.cat([dxq.to(dt), dxk.to(dt), s["dv"]], dim=1).flatten(1)
    return {"q": yq.to(dt), "k": yk.to(dt), "v": v.contiguous(), "dqkv": dqkv, "dwq": dwq, "dwk": dwk}


def _token_places(s, total):
    """Sequence and position of every new token (padding behind the last sequence left out)."""
    cu = s["cu_q"].long()
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return b, s["seq_lens"].long()[b] - (cu[b + 1] - t)


def _pages(x, head_major):
    return x.transpose(1, 2) if head_major else x


def _plain_append(s):
    dt, c = s["qkv"].dtype, s["case"]
    n = s["qkv"].shape[0] - c["pad"]
    b, pos = _token_places(s, n)
    cs = _turn(s, pos)
    q, k, v = _heads(s, s["qkv"][:n])
    yq, yk = (_rotate(s, x if w is None else x * w, cs) for x, w in (
        (_normed(q.float(), s.get("wq"))[0], s.get("wq")), (_normed(k.float(), s.get("wk"))[0], s.get("wk"))))
    s["out"][:n] = yq.to(dt)
    where = s["table"].long()[b, pos // c["page"]], pos % c["page"]
    _pages(s["keys"], c["head_major"])[where] = yk.to(dt)
    _pages(s["values"], c["head_major"])[where] = v
    return {"q": s["out"], "keys": s["keys"], "values": s["values"]}


def _attend(s, wide):
    """The padded batch: scores of all (query, key) pairs, masked, in ``wide``."""
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    n = s["q"].shape[0] - c["pad"]
    cu, lens = s["cu_q"].long(), s["seq_lens"].long()
    qlen = cu[1:] - cu[:-1]
    sm, tm = c["kv_hi"], c["q_hi"]
    rows = [_pages(x, c["head_major"])[s["table"].long().clamp(min=0)].flatten(1, 2)[:, :sm].to(wide)
            for x in (s["keys"], s["values"])]
    k, v = (x.permute(0, 2, 1, 3) for x in rows)  # [B, Hk, S, D]
    t = torch.arange(tm, device="cuda")
    idx = (cu[:-1, None] + t[None]).clamp(max=max(n - 1, 0))
    q = s["q"][idx].to(wide).view(len(lens), tm, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).view(len(lens), hk, h // hk, tm, k.shape[2])
    scores *= d ** -0.5
    last = (lens - qlen)[:, None] + t[None]  # the last key of each query
    j = torch.arange(k.shape[2], device="cuda")
    dead = (j[None, None] > last[:, :, None]) | (j[None, None] >= lens[:, None, None])
    scores.masked_fill_(dead[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.exp_()
    den = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).view(len(lens), hk, h // hk, tm, d)
    o = torch.where(den > 0, o / den, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    b, pos = _token_places(s, n)
    return o[b, torch.arange(n, device="cuda") - cu[b]]


def _plain_attention(s):
    o = _attend(s, torch.float32)
    s["out"][: o.shape[0]] = o.to(s["out"].dtype)
    return {"o": s["out"]}


def _controlled(s, wide):
    v = s["case"]["vocab"]
    x = s["logits"].to(wide)
    b, n = s["history"].shape
    at = torch.arange(n, device="cuda")[None]
    seen = torch.zeros(b, v, device="cuda", dtype=torch.int32)
    made = torch.zeros(b, v, device="cuda", dtype=torch.int32)
    ids = s["history"].long()
    seen.scatter_add_(1, ids, (at < s["history_len"][:, None]).int())
    made.scatter_add_(1, ids, ((at < s["history_len"][:, None]) & (at >= s["prompt_len"][:, None])).int())
    rep = s["repetition"].to(wide)[:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"].to(wide)[:, None] * made - s["presence"].to(wide)[:, None] * (made > 0)
    if "bias_ids" in s:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"].to(wide))
    if "mask" in s:
        t = torch.arange(v, device="cuda")
        allowed = (s["mask"][:, t // 32] >> (t % 32).int()[None]) & 1
        x = x.masked_fill(allowed == 0, -math.inf)
    return x


# ---- the framework's calls ------------------------------------------------------------------------------------


def _own_views(s):
    """The state's tensors as the framework's arrays (the handles a program keeps)."""
    from minifield_training_b200.device import DeviceArray
    from minifield_training_b200.kernels.paged import PagedCache

    def view(x, dtype=None):
        if x is None:
            return None
        dtype = dtype or {torch.int32: "int32", torch.float32: "float32"}.get(x.dtype) or s["name"]
        return DeviceArray(tuple(x.shape), dtype, ptr=x.data_ptr(), owner=False)

    o = {k: view(x) for k, x in s.items() if isinstance(x, torch.Tensor)}
    if "outs" in s:
        o["outs"], o["dw"] = [view(x) for x in s["outs"]], [view(x) for x in s["dw"]]
    if "keys" in s:
        o["cache"] = PagedCache(o["keys"], o["values"], head_major=s["case"]["head_major"])
    return o


def _own(s):
    from minifield_training_b200.kernels import logits, paged, rotary

    o = s.get("own")
    if o is None:
        o = s["own"] = _own_views(s)
    c, stream = s["case"], torch.cuda.current_stream().cuda_stream or None
    if c["op"] == "logits":
        logits.process_logits(o["logits"], history=o["history"], prompt_len=o["prompt_len"],
                              history_len=o["history_len"], repetition=o["repetition"], frequency=o["frequency"],
                              presence=o["presence"], bias_ids=o.get("bias_ids"), bias_values=o.get("bias_values"),
                              mask=o.get("mask"), out=o["out"], stream=stream)
        return {"logits": s["out"]}
    if c["op"] == "attention":
        paged.paged_attention(o["q"], o["cache"], o["cu_q"], o["seq_lens"], o["table"], max_q=s["max_q"],
                              out=o["out"], stream=stream)
        return {"o": s["out"]}
    turn = dict(interleaved=c["interleaved"], amplitude=s["amplitude"], q_weight=o.get("wq"), k_weight=o.get("wk"),
                eps=EPS, stream=stream)
    if c["op"] == "append":
        paged.paged_append(o["qkv"], o["cache"], o["cu_q"], o["seq_lens"], o["table"], heads=c["heads"],
                           freqs=o["freqs"], out=o["out"], **turn)
        return {"q": s["out"], "keys": s["keys"], "values": s["values"]}
    q, k, v, dqkv = o["outs"]
    rotary.qk_rotary_fwd(o["qkv"], o["positions"], o["freqs"], heads=c["heads"], kv_heads=c["kv_heads"],
                         out=(q, k, v), **turn)
    rotary.qk_rotary_bwd(o["qkv"], o["positions"], o["freqs"], o["dq"], o["dk"], o["dv"], out=dqkv,
                         weight_grads=tuple(o["dw"]) if c["norm"] else None, **turn)
    dw = s["dw"] if c["norm"] else [None, None]
    return {"q": s["outs"][0], "k": s["outs"][1], "v": s["outs"][2], "dqkv": s["outs"][3], "dwq": dw[0], "dwk": dw[1]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rotary":
        return _plain_rotary(state)
    if op == "append":
        return _plain_append(state)
    if op == "attention":
        return _plain_attention(state)
    state["out"].copy_(_controlled(state, torch.float32))
    return {"logits": state["out"]}


# ---- exact values ---------------------------------------------------------------------------------------------


def _exact_heads(s, x, positions, w, dy=None):
    """Rotation of normalised heads in float64 as complex products; with dy, the gradients too."""
    c, r = s["case"], s["rotary_dim"]
    x = x.double()
    angle = positions.double()[:, None, None] * s["freqs"].double()
    z = torch.polar(torch.full_like(angle, s["amplitude"]), angle)

    def spin(u, by):
        a, rest = u[..., :r], u[..., r:]
        pairs = a.unflatten(-1, (-1, 2)) if c["interleaved"] else a.unflatten(-1, (2, -1)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        y = y if c["interleaved"] else y.transpose(-1, -2)
        return torch.cat([y.flatten(-2), rest], dim=-1)

    gain = torch.ones(x.shape[-1], dtype=torch.float64, device="cuda") if w is None else w.double()
    norm = torch.ones_like(x[..., :1]) if w is None else ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
    y = spin(x / norm * gain, z)
    if dy is None:
        return y
    dn = spin(dy.double(), z.conj())
    if w is None:
        return y, dn, None
    d = x.shape[-1]
    dx = gain * dn / norm - x * (gain * dn * x).sum(-1, keepdim=True) / (d * norm ** 3)
    return y, dx, (dn * x / norm).sum((0, 1))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        b, v = s["logits"].shape
        x = s["logits"].cpu().numpy() if case["dtype"] != "bf16" else s["logits"].double().cpu().numpy()
        x = x.astype(np.float64)
        hist, used, prompt = (s[k].cpu().numpy() for k in ("history", "history_len", "prompt_len"))
        rep, freq, pres = (s[k].double().cpu().numpy() for k in ("repetition", "frequency", "presence"))
        for i in range(b):
            seen = np.unique(hist[i, : used[i]])
            x[i, seen] = np.where(x[i, seen] > 0, x[i, seen] / rep[i], x[i, seen] * rep[i])
            made, count = np.unique(hist[i, prompt[i]: used[i]], return_counts=True)
            x[i, made] -= freq[i] * count + pres[i]
            if "bias_ids" in s:
                x[i, s["bias_ids"][i].cpu().numpy()] += s["bias_values"][i].double().cpu().numpy()
            if "mask" in s:
                bits = np.unpackbits(s["mask"][i].cpu().numpy().view(np.uint8), bitorder="little")[:v]
                x[i, bits == 0] = -np.inf
        return {"logits": torch.from_numpy(x)}
    if op == "attention":
        c, o = s["case"], s["out"].double()
        cu, lens, page = s["cu_q"].tolist(), s["seq_lens"].tolist(), case["page"]
        h, hk = c["heads"], c["kv_heads"]
        for b, n in enumerate(lens):
            t = cu[b + 1] - cu[b]
            if not t:
                continue
            ids = s["table"][b, : -(-n // page)].long()
            k, v = (_pages(x[ids], c["head_major"]).flatten(0, 1)[:n].double() for x in (s["keys"], s["values"]))
            q = s["q"][cu[b]: cu[b + 1]].double() / math.sqrt(c["head_dim"])
            late = torch.ones(t, n, dtype=torch.bool, device="cuda").triu(n - t + 1)
            for i in range(h):
                a = (q[:, i] @ k[:, i * hk // h].T).masked_fill_(late, -math.inf)
                o[cu[b]: cu[b + 1], i] = torch.softmax(a, -1) @ v[:, i * hk // h]
        return {"o": o}
    if op == "append":
        n = s["qkv"].shape[0] - case["pad"]
        cu, lens = s["cu_q"].tolist(), s["seq_lens"].tolist()
        seq = [b for b in range(len(lens)) for _ in range(cu[b + 1] - cu[b])]
        pos = [lens[b] - cu[b + 1] + i for i, b in enumerate(seq)]
        p, q = torch.tensor(pos, device="cuda"), s["out"].double()
        hq, hkk, hv = _heads(s, s["qkv"][:n])
        q[:n] = _exact_heads(s, hq, p, s.get("wq"))
        keys, values = s["keys"].double(), s["values"].double()
        at = s["table"].long()[torch.tensor(seq, device="cuda"), p // case["page"]], p % case["page"]
        _pages(keys, case["head_major"])[at] = _exact_heads(s, hkk, p, s.get("wk"))
        _pages(values, case["head_major"])[at] = hv.double()
        return {"q": q, "keys": keys, "values": values}
    hq, hkk, hv = _heads(s, s["qkv"])
    yq, dxq, dwq = _exact_heads(s, hq, s["positions"], s.get("wq"), s["dq"])
    yk, dxk, dwk = _exact_heads(s, hkk, s["positions"], s.get("wk"), s["dk"])
    dqkv = torch.cat([dxq, dxk, s["dv"].double()], dim=1).flatten(1)
    return {"q": yq, "k": yk, "v": hv.double(), "dqkv": dqkv, "dwq": dwq, "dwk": dwk}
