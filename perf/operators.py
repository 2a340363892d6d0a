"""The 8-bit decoder operators: what is measured, and their plain forms.

Five operators of a decoder layer on 8-bit weights and of its readout:
  quantize   activations to 8-bit floating point with a scale per 128 columns
  linear     the matrix product of 8-bit operands with a scale per block of 128
  norm       the norm after a block, its gate, the residual add and the next norm
  rotary     rotary positions on query and key heads
  logprobs   log probabilities of given tokens, entropy and top alternatives
Sizes are those of this repository's decoder presets and of its token counts
(one token, one decision of ~515 tokens, a batch of decisions).
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
AMAX_FLOOR = 1e-30
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1}
DEV = "cuda"


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One new token's hidden state on its way into a projection.
        dict(name="quantize one token", op="quantize", rows=1, cols=4096, dtype="bf16", gated=False),
        # A prefill batch's gate and up columns (one [rows, 2 * cols] product) into the down projection's operand.
        dict(name="quantize gated prefill", op="quantize", rows=8192, cols=12288, dtype="fp16", gated=True),
        # One token's query / key / value projection: the weights are read for a single row.
        dict(name="linear one token", op="linear", rows=1, n=6144, k=4096, dtype="bf16", bias=False),
        # The down projection of 37 sequences that each add one token.
        dict(name="linear few rows", op="linear", rows=37, n=4096, k=12288, dtype="fp16", bias=False),
        # One decision's tokens through the query / key / value projection of a model with biases.
        dict(name="linear one decision", op="linear", rows=515, n=6144, k=4096, dtype="bf16", bias=True),
        # A batch of decisions through the gate / up projection.
        dict(name="linear prefill", op="linear", rows=8192, n=24576, k=4096, dtype="bf16", bias=False),
        # One token between two blocks, with a layer scale.
        dict(name="norm one token", op="norm", rows=1, cols=4096, dtype="bf16", res="fp32", gate="channel", out="bf16",
             post=True, pre=True),
        # A prefill batch between two blocks, straight into the next projection's 8-bit operand.
        dict(name="norm prefill", op="norm", rows=16384, cols=4096, dtype="bf16", res="fp32", gate="channel", out="fp8",
             post=True, pre=True),
        # One token far into a long context.
        dict(name="rotary one token", op="rotary", rows=1, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             layout="half", scaling="yarn", max_pos=131072, dtype="bf16"),
        # A prefill batch, a quarter of each head rotated, heads read out of the packed projection.
        dict(name="rotary prefill", op="rotary", rows=16384, heads=16, kv_heads=4, head_dim=256, rotary_dim=64,
             layout="interleaved", scaling="none", max_pos=8192, dtype="fp16"),
        # The next token's alternatives.
        dict(name="logprobs one token", op="logprobs", rows=1, vocab=152064, dtype="bf16", targets=1, top=20,
             temperature=1.0, masked=False),
        # Candidate answers scored over a batch, part of the rows restricted to the option labels.
        dict(name="logprobs batch", op="logprobs", rows=1024, vocab=256000, dtype="bf16", targets=4, top=8,
             temperature=0.7, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "norm", "rotary", "logprobs"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "quantize":
        cols = rng.choice([768, 2048, 4096, 5120, 12288, _log(rng, 64, 12288)])
        return dict(op=op, rows=_log(rng, 1, 8192), cols=cols, dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    gated=rng.random() < 0.5)
    if op == "linear":
        n = rng.choice([4096, 5120, 6144, 16384, 24576, _log(rng, 128, 24576)])
        k = rng.choice([2048, 4096, _log(rng, 64, 4096)])
        if rng.random() < 0.3:
            n, k = rng.choice([(4096, 12288), (2048, 16384), (_log(rng, 128, 4096), _log(rng, 4096, 16384))])
        return dict(op=op, rows=_log(rng, 1, 8192), n=n, k=k, dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]),
                    bias=rng.random() < 0.5)
    if op == "norm":
        cols = rng.choice([768, 2048, 4096, 5120, _log(rng, 64, 5120)])
        post = rng.random() < 0.7
        return dict(op=op, rows=_log(rng, 1, 12288), cols=cols, dtype=dtype, res=rng.choice(["fp32", "fp32", dtype]),
                    gate=rng.choice(["none", "channel", "row", "full"]), out=rng.choice(["fp8", dtype]), post=post,
                    pre=not post or rng.random() < 0.8)
    if op == "rotary":
        heads, kv_heads, hd = rng.choice([(32, 8, 128), (40, 8, 128), (8, 1, 256), (16, 4, 256), (12, 12, 64)])
        return dict(op=op, rows=_log(rng, 1, 12288), heads=heads, kv_heads=kv_heads, head_dim=hd,
                    rotary_dim=rng.choice([hd, hd, hd // 2, hd // 4]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "yarn", "llama3"]), max_pos=_log(rng, 512, 262144),
                    dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]))
    return dict(op=op, rows=_log(rng, 1, 512), vocab=rng.choice([50368, 152064, 250002, _log(rng, 1000, 256000)]),
                dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), targets=rng.randint(1, 8), top=rng.randint(0, 20),
                temperature=rng.choice([1.0, 0.5, 1.7]), masked=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(g, rows, cols):
    """Hidden-state-like values: unit normal rows of differing size, a few large channels."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    big = torch.rand(cols, generator=g, device=DEV) < 0.005
    return x * torch.where(big, 12.0, 1.0)


def _pad16(n):
    return (n + 15) // 16 * 16


def _to_f8(v, amax):
    inv = F8_MAX / amax
    return (v * inv).clamp(-F8_MAX, F8_MAX).to(F8), amax / F8_MAX


def _blocks(v):
    """[rows, cols] -> [rows, ceil(cols / 128), 128], zero-padded."""
    rows, cols = v.shape
    nb = -(-cols // 128)
    if nb * 128 != cols:
        v = torch.nn.functional.pad(v, (0, nb * 128 - cols))
    return v.view(rows, nb, 128)


def _plain_quantize(v):
    rows, cols = v.shape
    b = _blocks(v)
    q, s = _to_f8(b, b.abs().amax(-1, keepdim=True).clamp_min(AMAX_FLOOR))
    return q.view(rows, -1)[:, :cols], s.view(rows, -1)


def _rows16(q):
    """The same 8-bit matrix with rows that start on 16 bytes, as the operators hold it."""
    rows, cols = q.shape
    buf = torch.zeros(rows, _pad16(cols), dtype=torch.uint8, device=DEV)
    buf[:, :cols] = q.view(torch.uint8) if q.is_contiguous() else q.contiguous().view(torch.uint8)
    return buf.view(F8)[:, :cols]


def _weight_f8(w):
    n, k = w.shape
    nb, kb = -(-n // 128), -(-k // 128)
    p = torch.nn.functional.pad(w, (0, kb * 128 - k, 0, nb * 128 - n)).view(nb, 128, kb, 128)
    q, s = _to_f8(p, p.abs().amax((1, 3), keepdim=True).clamp_min(AMAX_FLOOR))
    return _rows16(q.reshape(nb * 128, kb * 128)[:n, :k]), s.view(nb, kb)


def _scaling(case):
    return {
        "none": None,
        "linear": {"type": "linear", "factor": 4.0},
        "yarn": {"type": "yarn", "factor": 8.0, "original_max_position": 16384, "beta_fast": 32.0, "beta_slow": 1.0},
        "llama3": {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                   "original_max_position": 8192},
    }[case["scaling"]]


THETA = 1e6


def _frequencies(case):
    """(radians per position in 64 bits [rotary_dim / 2], factor on the rotated values)."""
    rd, s = case["rotary_dim"], _scaling(case)
    i = torch.arange(0, rd, 2, dtype=torch.float64)
    f = THETA ** (-i / rd)
    if s is None:
        return f, 1.0
    if s["type"] == "linear":
        return f / s["factor"], 1.0
    if s["type"] == "yarn":
        def dim(turns):
            return rd * math.log(s["original_max_position"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        lo, hi = max(math.floor(dim(s["beta_fast"])), 0), min(math.ceil(dim(s["beta_slow"])), rd - 1)
        ramp = ((torch.arange(rd // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / s["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(s["factor"]) + 1.0
    wave = 2 * math.pi / f
    lo, hi, orig = s["low_freq_factor"], s["high_freq_factor"], s["original_max_position"]
    t = ((orig / wave - lo) / (hi - lo)).clamp(0, 1)
    return (1 - t) * f / s["factor"] + t * f, 1.0


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"case": case}
    if op == "quantize":
        t = TYPES[case["dtype"]]
        rows, cols = case["rows"], case["cols"]
        if case["gated"]:
            both = _activations(g, rows, 2 * cols).to(t)
            st["gate"], st["x"] = both[:, :cols], both[:, cols:]
        else:
            st["gate"], st["x"] = None, _activations(g, rows, cols).to(t)
    elif op == "linear":
        q, st["a_scale"] = _plain_quantize(_activations(g, case["rows"], case["k"]))
        st["a"] = _rows16(q)
        st["w"], st["w_scale"] = _weight_f8(torch.randn(case["n"], case["k"], generator=g, device=DEV) * case["k"] ** -0.5)
        st["bias"] = torch.randn(case["n"], generator=g, device=DEV) * 0.1 if case["bias"] else None
    elif op == "norm":
        rows, cols = case["rows"], case["cols"]
        st["y"] = (3.0 * _activations(g, rows, cols)).to(TYPES[case["dtype"]])
        st["h"] = (4.0 * _activations(g, rows, cols)).to(TYPES[case["res"]])
        gain = lambda: 1.0 + 0.2 * torch.randn(cols, generator=g, device=DEV)  # noqa: E731
        st["post"] = gain() if case["post"] else None
        st["pre"] = gain() if case["pre"] else None
        shape = {"none": None, "channel": (cols,), "row": (rows, 1), "full": (rows, cols)}[case["gate"]]
        st["gate"] = None
        if shape:
            gate = 0.5 + 0.1 * torch.randn(*shape, generator=g, device=DEV)
            st["gate"] = gate if case["gate"] == "channel" else gate.to(TYPES[case["dtype"]])
    elif op == "rotary":
        rows, h, kv, hd = case["rows"], case["heads"], case["kv_heads"], case["head_dim"]
        qkv = torch.randn(rows, (h + 2 * kv) * hd, generator=g, device=DEV).to(TYPES[case["dtype"]])
        st["q"] = qkv[:, :h * hd].view(rows, h, hd)
        st["k"] = qkv[:, h * hd:(h + kv) * hd].view(rows, kv, hd)
        # Sequences of a packed batch: each starts somewhere in the context and runs on.
        start = torch.randint(0, case["max_pos"], (rows,), generator=g, device=DEV, dtype=torch.int64)
        idx = torch.arange(rows, device=DEV)
        st["positions"] = ((start[(idx // 512) * 512] + idx % 512) % case["max_pos"]).to(torch.int32)
        if own:
            from verdict_b200 import ops
            st["plan"] = ops.RotaryPlan(hd, rotary_dim=case["rotary_dim"], theta=THETA, scaling=_scaling(case),
                                        layout=case["layout"])
        else:
            f, m = _frequencies(case)
            ang = torch.arange(case["max_pos"], device=DEV, dtype=torch.float64)[:, None] * f.to(DEV)[None]
            st["cos"], st["sin"] = (ang.cos() * m).float(), (ang.sin() * m).float()
    else:
        rows, v, t = case["rows"], case["vocab"], TYPES[case["dtype"]]
        x = torch.empty(rows, v, device=DEV, dtype=t)
        for r in range(0, rows, 256):
            c = torch.randn(min(256, rows - r), v, generator=g, device=DEV)
            x[r:r + 256] = (c * torch.empty(c.shape[0], 1, device=DEV).uniform_(1.0, 4.0, generator=g)).to(t)
        ids = torch.randint(0, v, (rows, case["targets"]), generator=g, device=DEV)
        if case["masked"]:
            # Every other row keeps a few hundred labels; the first row of a longer batch keeps none.
            live = torch.randint(0, v, (min(255, v),), generator=g, device=DEV)
            keep = torch.zeros(v, dtype=torch.bool, device=DEV)
            keep[live] = True
            x[1::2] = torch.where(keep, x[1::2], torch.tensor(-math.inf, dtype=t, device=DEV))
            ids[1::2] = live[ids[1::2] % live.numel()]
            if rows > 2:
                x[0] = -math.inf
        st["logits"], st["ids"] = x, ids
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from verdict_b200 import ops
    case = st["case"]
    op = case["op"]
    if op == "quantize":
        q, s = ops.quantize_fp8(st["x"], gate=st["gate"], act="silu" if case["gated"] else "none")
        return {"q": q, "scale": s}
    if op == "linear":
        return {"out": ops.fp8_linear(st["a"], st["a_scale"], st["w"], st["w_scale"], bias=st["bias"],
                                      out_dtype=TYPES[case["dtype"]])}
    if op == "norm":
        out = None if not case["pre"] else F8 if case["out"] == "fp8" else TYPES[case["out"]]
        r = ops.block_norm(st["y"], st["h"], post_gain=st["post"], gate=st["gate"], residual_scale=RES_SCALE,
                           block_scale=BLOCK_SCALE, pre_gain=st["pre"], eps=EPS, out_dtype=out)
        d = {"h": r.residual}
        if case["pre"]:
            d["z"] = r.out
            if case["out"] == "fp8":
                d["scale"] = r.scale
        return d
    if op == "rotary":
        q, k = ops.rotary(st["q"], st["k"], st["positions"], st["plan"])
        return {"q": q, "k": k}
    r = ops.token_logprobs(st["logits"], st["ids"], top=case["top"], temperature=case["temperature"])
    d = {"logprobs": r.logprobs, "entropy": r.entropy, "lse": r.lse}
    if case["top"]:
        d["top_ids"], d["top_logprobs"] = r.top_ids, r.top_logprobs
    return d


EPS = 1e-6
RES_SCALE = 0.9
BLOCK_SCALE = 0.7


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _rotate(x, cos, sin, layout):
    rd = 2 * cos.shape[-1]
    r, rest = x[..., :rd].float(), x[..., rd:]
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = r[..., :rd // 2], r[..., rd // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([r.to(x.dtype), rest], -1)


def _order_keys(x):
    """int64 keys that sort like (value, then lowest index first); all distinct within a row."""
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
    return b * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "quantize":
        v = st["x"].float()
        if case["gated"]:
            gate = st["gate"].float()
            v = gate / (1 + torch.exp(-gate)) * v
        q, s = _plain_quantize(v)
        return {"q": q, "scale": s}
    if op == "linear":
        n, k = st["w"].shape
        a = st["a"].float() * st["a_scale"].repeat_interleave(128, 1)[:, :k]
        w = st["w"].float() * st["w_scale"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        out = torch.matmul(a, w.T)
        if st["bias"] is not None:
            out += st["bias"]
        return {"out": out.to(TYPES[case["dtype"]])}
    if op == "norm":
        u = st["y"].float()
        if case["post"]:
            u = _rms(u) * st["post"]
        if st["gate"] is not None:
            u = u * st["gate"].float()
        h = RES_SCALE * st["h"].float() + BLOCK_SCALE * u
        d = {"h": h.to(st["h"].dtype)}
        if case["pre"]:
            z = _rms(h) * st["pre"]
            if case["out"] == "fp8":
                d["z"], d["scale"] = _plain_quantize(z)
            else:
                d["z"] = z.to(TYPES[case["out"]])
        return d
    if op == "rotary":
        at = st["positions"].long()
        cos, sin = st["cos"][at], st["sin"][at]
        return {"q": _rotate(st["q"], cos, sin, case["layout"]), "k": _rotate(st["k"], cos, sin, case["layout"])}
    x = st["logits"].float()
    top = x.amax(-1, keepdim=True)
    empty = top == -math.inf
    z = (x - top.masked_fill(empty, 0.0)) / case["temperature"]
    e = torch.exp(z)
    s = e.sum(-1, keepdim=True)
    log_s = torch.log(s)
    d = {"logprobs": torch.where(empty, -math.inf, z.gather(1, st["ids"]) - log_s),
         "entropy": torch.where(empty, 0.0, log_s - (e * z.masked_fill(e == 0, 0.0)).sum(-1, keepdim=True) / s)[:, 0],
         "lse": (top / case["temperature"] + log_s)[:, 0]}
    if case["top"]:
        at = torch.topk(_order_keys(x), case["top"], dim=-1).indices
        lp = torch.where(empty, -math.inf, z.gather(1, at) - log_s)
        d["top_ids"] = torch.where(x.gather(1, at) == -math.inf, -1, at).to(torch.int32)
        d["top_logprobs"] = lp
    return d


# ---------------------------------------------------------------------------
# Work and the answers in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "quantize":
        m, k = case["rows"], case["cols"]
        n_in = 2 if case["gated"] else 1
        return {"bytes": m * k * (n_in * BYTES[case["dtype"]] + 1) + 4 * m * -(-k // 128), "flops": m * k * (2 + 5 * (n_in - 1))}
    if op == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        kb = -(-k // 128)
        return {"bytes": m * k + n * k + 4 * (m + -(-n // 128)) * kb + m * n * BYTES[case["dtype"]] + 4 * n * case["bias"],
                "flops": 2 * m * n * k}
    if op == "norm":
        m, d = case["rows"], case["cols"]
        gate = {"none": 0, "channel": 4 * d, "row": m * BYTES[case["dtype"]], "full": m * d * BYTES[case["dtype"]]}[case["gate"]]
        b = m * d * (BYTES[case["dtype"]] + 2 * BYTES[case["res"]]) + gate + 4 * d * (case["post"] + case["pre"])
        if case["pre"]:
            b += m * d * BYTES[case["out"]] + (4 * m * -(-d // 128) if case["out"] == "fp8" else 0)
        return {"bytes": b, "flops": 10 * m * d}
    if op == "rotary":
        el = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * el * case["head_dim"] * BYTES[case["dtype"]] + 4 * case["rows"], "flops": 3 * el * case["rotary_dim"]}
    t, v = case["rows"], case["vocab"]
    return {"bytes": t * v * BYTES[case["dtype"]] + t * (12 * case["targets"] + 8 * case["top"] + 8), "flops": 4 * t * v}


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    D = torch.float64
    if op == "quantize":
        v = st["x"].to(D)
        if case["gated"]:
            v = v * st["gate"].to(D) * torch.sigmoid(st["gate"].to(D))
        scale = [c.abs().amax(1).clamp_min(AMAX_FLOOR) / F8_MAX for c in v.split(128, 1)]
        return {"q": None, "scale": torch.stack(scale, 1)}
    if op == "linear":
        n, k = st["w"].shape
        out = torch.zeros(case["rows"], n, dtype=D, device=DEV)
        col = torch.arange(n, device=DEV) // 128
        for b, k0 in enumerate(range(0, k, 4096)):
            kk = torch.arange(k0, min(k0 + 4096, k), device=DEV)
            a = st["a"].view(torch.uint8)[:, kk].view(F8).to(D) * st["a_scale"].to(D)[:, kk // 128]
            w = st["w"].view(torch.uint8)[:, kk].view(F8).to(D) * st["w_scale"].to(D)[col][:, kk // 128]
            out += a @ w.T
        return {"out": out + st["bias"].to(D) if case["bias"] else out}
    if op == "norm":
        def normed(t, gain):
            return t / (t.pow(2).mean(1, keepdim=True) + EPS).sqrt() * gain.to(D)
        u = st["y"].to(D)
        u = normed(u, st["post"]) if case["post"] else u
        h = st["h"].to(D) * RES_SCALE + u * BLOCK_SCALE * (1.0 if st["gate"] is None else st["gate"].to(D))
        d = {"h": h}
        if case["pre"]:
            z = normed(h, st["pre"])
            if case["out"] == "fp8":
                d["z"] = None
                d["scale"] = torch.stack([c.abs().amax(1).clamp_min(AMAX_FLOOR) / F8_MAX for c in z.split(128, 1)], 1)
            else:
                d["z"] = z
        return d
    if op == "rotary":
        f, m = _frequencies(case)
        ang = st["positions"].to(D)[:, None, None] * f.to(DEV)
        turn = torch.polar(torch.full_like(ang, m), ang)
        rd, half = case["rotary_dim"], case["rotary_dim"] // 2
        d = {}
        for name in ("q", "k"):
            x = st[name].to(D)
            if case["layout"] == "half":
                c = torch.complex(x[..., :half], x[..., half:rd]) * turn
                r = torch.cat([c.real, c.imag], -1)
            else:
                r = torch.view_as_real(torch.complex(x[..., 0:rd:2], x[..., 1:rd:2]) * turn).flatten(-2)
            d[name] = torch.cat([r, x[..., rd:]], -1)
        return d
    lp, ent, lse, tops = [], [], [], []
    for r in range(0, case["rows"], 64):
        x = st["logits"][r:r + 64].to(D) / case["temperature"]
        norm = torch.logsumexp(x, 1, keepdim=True)
        dead = norm == -math.inf
        p = x - torch.where(dead, 0.0, norm)
        lp.append(p.gather(1, st["ids"][r:r + 64]))
        ent.append(torch.special.entr(torch.where(dead, 0.0, p.exp())).sum(1))
        lse.append(norm[:, 0])
        tops.append(p.topk(case["top"], 1).values)
    d = {"logprobs": torch.cat(lp), "entropy": torch.cat(ent), "lse": torch.cat(lse)}
    if case["top"]:
        d["top_ids"], d["top_logprobs"] = None, torch.cat(tops)
    return d
