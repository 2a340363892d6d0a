"""The 8-bit decoder operators (verdict_b200/ops.py) against their definitions in 64 bits.

Tolerances, from the number formats and the operators' sums:
- u = 2^-24 is fp32's rounding; a 16-bit output adds half a unit in its last
  place, relative 2^-11 (fp16, 11 significant bits; 2^-25 absolute below its
  smallest normal number) or 2^-8 (bf16, 8 significant bits);
- e4m3 rounds to within 2^-4 of a value, or 2^-10 of the scale below its
  smallest normal number;
- a sum of n fp32 terms is within n u of the sum of their magnitudes.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import _abi, ops  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: U}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-30, torch.float32: 1e-30}
F8 = torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, ref, bound):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[~finite & ~torch.isnan(ref)], ref[~finite & ~torch.isnan(ref)])
    err = torch.where(finite, (got - torch.where(finite, ref, 0.0)).abs(), 0.0)
    bad = finite & ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {ref.numel()} off, worst {float((err / bound)[bad].max()):.3g} x bound"


def strided(t, pad, offset=0):
    """The same matrix as a view of a wider buffer, `offset` elements into each row."""
    buf = torch.full((t.shape[0], offset + t.shape[1] + pad), math.nan, device="cuda").to(t.dtype)
    view = buf[:, offset:offset + t.shape[1]]
    view.copy_(t)
    return view


def blocks_of(v, fn):
    return torch.stack([fn(c) for c in v.split(128, 1)], 1)


def dequant(q, scale):
    return q.double() * scale.double().repeat_interleave(128, 1)[:, :q.shape[1]]


# ---------------------------------------------------------------------------
# Casts
# ---------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 128), (3, 127), (5, 129), (2, 520), (37, 4096), (300, 12288), (0, 128)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_quantize_is_the_rounded_definition(rows, cols, dt):
    x = randn(gen(rows + cols), rows, cols, dtype=DT[dt], scale=3.0)
    for view in (x, strided(x, 5), strided(x, 8, 3)):
        q, s = ops.quantize_fp8(view)
        assert q.dtype == F8 and q.shape == x.shape and s.shape == (rows, -(-cols // 128))
        if rows == 0:
            continue
        amax = blocks_of(x.float(), lambda c: c.abs().amax(1)).clamp_min(1e-30)
        c448 = torch.full_like(amax, 448.0)
        assert torch.equal(s, amax / c448)
        inv = (c448 / amax).repeat_interleave(128, 1)[:, :cols]
        want = (x.float() * inv).clamp(-448, 448).to(F8)
        assert torch.equal(q.float(), want.float())


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu", "none"])
@pytest.mark.parametrize("rows,cols", [(1, 130), (65, 1024)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_quantize_gated(rows, cols, act, dt):
    g = gen(cols)
    both = randn(g, rows, 2 * cols, dtype=DT[dt], scale=2.0)
    gate, x = both[:, :cols], both[:, cols:]
    q, s = ops.quantize_fp8(x, gate=gate, act=act)
    f = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "none": lambda t: t,
         "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act]
    v = f(gate.double()) * x.double()
    # The activations carry a few fp32 roundings, gelu's erf 1.5e-7 absolute.
    slack = 1e-5 * (v.abs() + x.double().abs())
    amax = blocks_of(v, lambda c: c.abs().amax(1))
    within(s, amax / 448, 2e-5 * amax / 448 + 1e-5 * blocks_of(x.double(), lambda c: c.abs().amax(1)) / 448)
    sc = s.double().repeat_interleave(128, 1)[:, :cols]
    within(dequant(q, s), v, torch.maximum(v.abs() * 2.0 ** -4, sc * 2.0 ** -10) * (1 + 1e-3) + slack)


def test_quantize_special_blocks():
    x = randn(gen(1), 4, 512)
    x[0, :128] = 0.0
    x[1, 130] = math.inf
    x[2, 260] = math.nan
    x[3, 384:] = 1e-38
    x[3, :128] *= 1e37
    q, s = ops.quantize_fp8(x)
    assert (q[0, :128].float() == 0).all() and s[0, 0] == np.float32(1e-30) / np.float32(448)
    assert math.isinf(s[1, 1]) and math.isnan(s[2, 2])
    d = dequant(q, s)
    assert torch.isnan(d[1, 128:256]).all() and torch.isnan(d[2, 256:384]).all()
    assert torch.isfinite(d[1, :128]).all() and torch.isfinite(d[1, 256:]).all() and torch.isfinite(d[3]).all()
    assert (q[3, 384:].float() == 0).all()  # far below the floor
    xd = x[3, :128].double()
    within(d[3, :128], xd, xd.abs() * 2.0 ** -4 * 1.001 + float(s[3, 0]) * 2.0 ** -10)


@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (130, 257), (300, 1000)])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_quantize_weight(rows, cols, dt):
    w = randn(gen(rows), rows, cols, dtype=DT[dt])
    q, s = ops.quantize_fp8_weight(strided(w, 3))
    f = w.float()
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            b = f[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128]
            amax = b.abs().max()
            assert s[i, j] == amax / torch.tensor(448.0, device="cuda")
            want = (b * (torch.tensor(448.0, device="cuda") / amax)).clamp(-448, 448).to(F8)
            assert torch.equal(q[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].float(), want.float())


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------
def operand(g, rows, cols, row_block):
    """Random codes over the whole format with scales, on rows padded with NaN codes."""
    ld = (cols + 15) // 16 * 16 + 16
    codes = torch.randint(0, 256, (rows, ld), generator=g, device="cuda", dtype=torch.int16).to(torch.uint8)
    codes = torch.where((codes & 0x7F) == 0x7F, torch.zeros_like(codes), codes)
    codes[:, cols:] = 0x7F
    s = torch.exp(torch.randn(-(-rows // row_block), -(-cols // 128), generator=g, device="cuda")) * 1e-2
    return codes.view(F8)[:, :cols], s


def linear_ref(a, sa, w, sw, bias):
    n, k = w.shape
    ad = dequant(a, sa)
    wd = w.double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    ref, mag = ad @ wd.T, ad.abs() @ wd.abs().T
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    return ref, mag


# Sums: 128 products per block in the tensor core (truncated rather than rounded: 2 u), then a rounding per block,
# per CTA that shares K (at most 8) and for the scales and the bias.
def linear_bound(mag, ref, k, dtype):
    n = 2 * 128 + -(-k // 128) + 12
    return n * U * mag + (HALF_ULP[dtype] * ref.abs() if dtype != torch.float32 else 0) + TINY[dtype]


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 130, 127), (1, 256, 4096), (2, 1000, 129), (31, 257, 640), (32, 128, 128), (33, 129, 2048),
    (64, 4096, 1024), (65, 127, 300), (128, 128, 16), (129, 640, 5000), (257, 1000, 384), (500, 2056, 1152),
    (1100, 1300, 200), (2100, 4100, 520)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_linear(m, n, k, dt):
    g = gen(m * 31 + n * 7 + k)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    bias = randn(g, n) if (m + n) % 2 else None
    ref, mag = linear_ref(a, sa, w, sw, bias)
    out = ops.fp8_linear(a, sa, w, sw, bias=bias, out_dtype=DT[dt])
    ops.check_status()
    bound = linear_bound(mag, ref, k, DT[dt])
    if dt == "fp16":
        ref = torch.where(ref.abs() > 65504, torch.inf * ref.sign(), ref)
        bound = torch.where(ref.abs() > 65000, torch.inf, bound)
    within(out, ref, bound)


@pytest.mark.parametrize("m,n,k", [(3, 200, 256), (70, 200, 256), (700, 1032, 384)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 0), (5, 1)])
def test_linear_output_strides(m, n, k, pad, offset):
    g = gen(m + pad)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    ref, mag = linear_ref(a, sa, w, sw, None)
    buf = torch.full((m, offset + n + pad), 7.0, device="cuda", dtype=torch.bfloat16)
    out = buf[:, offset:offset + n]
    # Scales in any row stride too.
    assert ops.fp8_linear(a, strided(sa, 2), w, strided(sw, 3), out=out) is out
    within(out, ref, linear_bound(mag, ref, k, torch.bfloat16))
    assert (buf[:, :offset] == 7).all() and (buf[:, offset + n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(5, 300, 2048), (65, 300, 256), (600, 1100, 256)])
def test_linear_nonfinite_rows_stay_apart(m, n, k):
    g = gen(m)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    clean = ops.fp8_linear(a, sa, w, sw)
    sa2 = sa.clone()
    sa2[1, 0], sa2[2, -1] = math.nan, math.inf
    out = ops.fp8_linear(a, sa2, w, sw)
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[1] = keep[2] = False
    assert torch.equal(out[keep], clean[keep])
    assert torch.isnan(out[1]).all() and not torch.isfinite(out[2]).any()


@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (37, 1024, 8192), (515, 1024, 1024), (2048, 2048, 512)])
def test_linear_repeats_bit_for_bit(m, n, k):
    g = gen(3)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    first = ops.fp8_linear(a, sa, w, sw, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(ops.fp8_linear(a, sa, w, sw, out_dtype=torch.float32), first)


# ---------------------------------------------------------------------------
# Norms
# ---------------------------------------------------------------------------
def norm_ref(y, h, post, gate, rs, bs, pre, eps, plus_one):
    def rms(t, gain):
        gain = gain.double() + (1 if plus_one else 0)
        return t / (t.pow(2).mean(1, keepdim=True) + eps).sqrt() * gain

    u = y.double() if y is not None else 0.0
    if post is not None:
        u = rms(u, post)
    if gate is not None:
        u = u * gate.double()
    parts = ([rs * h.double()] if h is not None else []) + ([bs * u] if y is not None else [])
    new = sum(parts)
    mag = sum(p.abs() for p in parts)
    return new, mag, rms(new, pre) if pre is not None else None


# The statistic's relative error: cols fp32 terms summed by a thread and then in a tree, far below 2^-20; with the
# products around it 2^-19 is a bound with room.
NORM_REL = 2.0 ** -19


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 7), (3, 128), (5, 771), (4, 2049), (33, 4096), (3, 5120), (2, 16384)])
@pytest.mark.parametrize("dt,res", [("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32"), ("bf16", "bf16")])
@pytest.mark.parametrize("gate_kind", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("out", ["same", "fp8"])
def test_block_norm(rows, cols, dt, res, gate_kind, out):
    g = gen(rows * cols)
    y, h = randn(g, rows, cols, dtype=DT[dt], scale=3.0), randn(g, rows, cols, dtype=DT[res], scale=5.0)
    post, pre = 1 + randn(g, cols, scale=0.1), 1 + randn(g, cols, scale=0.1)
    shape = {"none": None, "channel": (cols,), "row": (rows, 1), "full": (rows, cols)}[gate_kind]
    gate = None if shape is None else randn(g, *shape, dtype=torch.float32 if gate_kind == "channel" else DT[dt])
    plus_one = cols % 2 == 1
    new, mag, z = norm_ref(y, h, post, gate, 0.9, 0.6, pre, 1e-6, plus_one)
    for yy, hh in ((y, h), (strided(y, 3), strided(h, 8))):
        r = ops.block_norm(yy, hh, post_gain=post, gate=gate, residual_scale=0.9, block_scale=0.6, pre_gain=pre,
                           plus_one=plus_one, out_dtype=F8 if out == "fp8" else None)
        assert r.residual.dtype == DT[res]
        within(r.residual, new, NORM_REL * mag + HALF_ULP[DT[res]] * new.abs() + TINY[DT[res]])
        # z's statistic and values both come from the new residual, whose error is relative to `mag`.
        zgain = (z / torch.where(new == 0, 1.0, new)).abs().amax(1, keepdim=True)
        zerr = 2 * NORM_REL * (z.abs() + mag * zgain)
        if out == "fp8":
            amax = blocks_of(z, lambda c: c.abs().amax(1))
            within(r.scale, amax / 448, (blocks_of(zerr, lambda c: c.amax(1)) + amax * 2 * U) / 448)
            sc = r.scale.double().repeat_interleave(128, 1)[:, :cols]
            within(dequant(r.out, r.scale), z,
                   torch.maximum(z.abs() * 2.0 ** -4, sc * 2.0 ** -10) * (1 + 1e-3) + 2 * zerr)
        else:
            assert r.scale is None and r.out.dtype == DT[dt]
            within(r.out, z, zerr + HALF_ULP[DT[dt]] * z.abs() + TINY[DT[dt]])


def test_block_norm_parts():
    g = gen(9)
    y, h = randn(g, 6, 300, dtype=torch.bfloat16), randn(g, 6, 300)
    pre = 1 + randn(g, 300, scale=0.1)
    # Only the norm before a block: the residual is handed through.
    r = ops.block_norm(None, h, pre_gain=pre, out_dtype=torch.bfloat16)
    _, _, z = norm_ref(None, h, None, None, 1.0, 1.0, pre, 1e-6, False)
    assert r.residual is h
    within(r.out, z, 4 * NORM_REL * z.abs() + HALF_ULP[torch.bfloat16] * z.abs())
    # Only the residual add; in place.
    h2 = h.clone()
    r = ops.block_norm(y, h2, block_scale=0.5, in_place=True)
    assert r.residual is h2 and r.out is None
    within(h2, h.double() + 0.5 * y.double(), 4 * U * (h.double().abs() + y.double().abs()))
    # No residual yet: the block's output starts one.
    r = ops.block_norm(y, None, pre_gain=pre)
    assert r.residual.dtype == torch.float32 and torch.equal(r.residual, y.float())
    # A gate broadcast from one row, and a zero one.
    r = ops.block_norm(y, h, gate=torch.zeros(1, 300, device="cuda"))
    assert torch.equal(r.residual, h)
    assert ops.block_norm(y[:0], h[:0], pre_gain=pre).out.shape == (0, 300)


def test_block_norm_zero_and_large_rows():
    y = torch.zeros(3, 256, device="cuda", dtype=torch.bfloat16)
    h = torch.zeros(3, 256, device="cuda")
    h[1] = 1e15
    h[2, 5] = math.nan
    one = torch.ones(256, device="cuda")
    r = ops.block_norm(y, h, post_gain=one, pre_gain=one, out_dtype=torch.float32)
    assert (r.out[0] == 0).all()
    within(r.out[1], torch.ones(256, device="cuda"), 1e-6)
    assert torch.isnan(r.out[2]).all()


# ---------------------------------------------------------------------------
# Rotary
# ---------------------------------------------------------------------------
def rotary_ref(x, pos, plan, inverse):
    rd = plan.rotary_dim
    # Angles from the plan's 64-bit turns with Python's integers: exact for any position.
    turns = [t % (1 << 64) for t in plan.turns.tolist()]
    frac = [[((p * t) % (1 << 64)) / 2.0 ** 64 for t in turns] for p in pos]
    ang = 2 * math.pi * torch.tensor(frac, dtype=torch.float64, device="cuda").reshape(len(pos), 1, rd // 2)
    c, s = ang.cos() * plan.factor, ang.sin() * plan.factor * (-1 if inverse else 1)
    x = x.double()
    if plan.interleaved:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        mag = torch.stack([a.abs() + b.abs()] * 2, -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
        mag = torch.cat([a.abs() + b.abs()] * 2, -1)
    return torch.cat([r, x[..., rd:]], -1), torch.cat([mag, torch.zeros_like(x[..., rd:])], -1)


# Cosine and sine: the angle carries 2^-24 of half a turn (pi u), the functions two units in the last place.
def rotary_bound(ref, mag, plan, dtype):
    return 8 * U * plan.factor * mag + (HALF_ULP[dtype] * ref.abs() if dtype != torch.float32 else 0) + TINY[dtype]


@pytest.mark.parametrize("hd,rd,heads,kv", [(128, 128, 4, 2), (64, 64, 3, 3), (256, 64, 2, 1), (128, 96, 1, 1),
                                            (10, 6, 2, 1), (80, 20, 2, 2), (128, 2, 2, 1)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_rotary(hd, rd, heads, kv, layout, dt):
    g = gen(hd + rd)
    plan = ops.RotaryPlan(hd, rotary_dim=rd, theta=1e4, layout=layout)
    for tokens in (1, 3, 9):
        qkv = randn(g, tokens, (heads + 2 * kv) * hd, dtype=DT[dt])
        q = qkv[:, :heads * hd].view(tokens, heads, hd)
        k = qkv[:, heads * hd:(heads + kv) * hd].view(tokens, kv, hd)
        pos = torch.randint(-5, 100000, (tokens,), generator=g, device="cuda")
        for p in (pos, pos.to(torch.int32)):
            qo, ko = ops.rotary(q, k, p, plan)
            for o, x in ((qo, q), (ko, k)):
                ref, mag = rotary_ref(x, pos.tolist(), plan, False)
                within(o, ref, rotary_bound(ref, mag, plan, DT[dt]))
                assert torch.equal(o[..., rd:], x[..., rd:])
        # Back again, in place, by itself.
        ref, mag = rotary_ref(qo, pos.tolist(), plan, True)
        ops.rotary(qo, None, pos, plan, inverse=True, q_out=qo)
        within(qo, ref, rotary_bound(ref, mag, plan, DT[dt]))


@pytest.mark.parametrize("scaling", [
    None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
    {"type": "yarn", "factor": 4.0, "original_max_position": 4096},
    {"type": "llama3", "factor": 8.0, "original_max_position": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
    {"type": "divisors", "divisors": [1.0 + i / 8 for i in range(32)], "attention_factor": 1.2}])
def test_rotary_far_positions(scaling):
    plan = ops.RotaryPlan(64, theta=1e6, scaling=scaling)
    pos = [0, 1, 131071, (1 << 31) - 1, 1 << 40, -(1 << 40), (1 << 62) + 12345]
    q = randn(gen(4), len(pos), 2, 64)
    out, none = ops.rotary(q, None, torch.tensor(pos, device="cuda"), plan)
    assert none is None
    ref, mag = rotary_ref(q, pos, plan, False)
    within(out, ref, rotary_bound(ref, mag, plan, torch.float32))
    # Consecutive tokens from a first position.
    out2, _ = ops.rotary(q, None, 131071, plan)
    ref, mag = rotary_ref(q, [131071 + i for i in range(len(pos))], plan, False)
    within(out2, ref, rotary_bound(ref, mag, plan, torch.float32))


def test_rotary_head_strides():
    plan = ops.RotaryPlan(64)
    g = gen(8)
    base = randn(g, 3, 5, 64, dtype=torch.bfloat16)
    by_head = base.transpose(0, 1).contiguous().transpose(0, 1)  # [tokens, heads, hd] laid out head by head
    pos = torch.tensor([3, 1, 4], device="cuda")
    want, _ = ops.rotary(base, None, pos, plan)
    got, _ = ops.rotary(by_head, None, pos, plan, q_out=torch.empty_like(base))
    assert torch.equal(got, want)
    shared = base[:, :1].expand(3, 5, 64)  # one head read five times
    got, _ = ops.rotary(shared, None, pos, plan)
    assert torch.equal(got, want[:, :1].expand(3, 5, 64))
    assert ops.rotary(base[:0], None, pos[:0], plan)[0].shape == (0, 5, 64)


# ---------------------------------------------------------------------------
# Log probabilities
# ---------------------------------------------------------------------------
def check_logprobs(x, ids, top, temperature):
    r = ops.token_logprobs(x, ids, top=top, temperature=temperature)
    rows, vocab = x.shape
    z = x.double() / temperature
    m = z.amax(1, keepdim=True)
    empty = m == -math.inf
    m = torch.where(empty, 0.0, m)
    log_s = torch.logsumexp(z - m, 1, keepdim=True)  # beside the maximum: it can be the type's lowest value
    p = z - m - torch.where(empty, 0.0, log_s)
    lse = m + log_s
    # exp by ex2.approx (2 u on the result, u |z| on the argument), sums of at most vocab / 512 terms a thread and a
    # tree: the sum is within 2^-19; the maximum enters the lse with u |m|.
    bound = 2.0 ** -19 + 8 * U * (m.abs() + 1)
    within(r.lse[:, None], lse, bound)
    ent = torch.special.entr(torch.where(empty, 0.0, p.exp())).sum(1, keepdim=True)
    within(r.entropy[:, None], ent, 4 * bound * (1 + ent))
    if ids is not None:
        within(r.logprobs, p.gather(1, ids), bound + 8 * U * p.gather(1, ids).nan_to_num(0, 0, 0).abs())
    if top:
        order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True)
        want = order.indices[:, :top]
        live = order.values[:, :top] > -math.inf
        want = torch.where(live, want, -1)
        lp = torch.where(live, p.gather(1, want.clamp_min(0)), -math.inf)
        if vocab < top:
            want = torch.nn.functional.pad(want, (0, top - vocab), value=-1)
            lp = torch.nn.functional.pad(lp, (0, top - vocab), value=-math.inf)
        assert torch.equal(r.top_ids.long(), want)
        within(r.top_logprobs, lp, bound + 8 * U * lp.nan_to_num(0, 0, 0).abs())
    return r


@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 7), (3, 8), (1, 1000), (5, 4097), (2, 32771), (300, 1024),
                                        (1, 152064), (40, 50368), (160, 9001)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("top,temperature", [(0, 1.0), (1, 0.3), (20, 1.0), (64, 2.0)])
def test_logprobs(rows, vocab, dt, top, temperature):
    g = gen(rows + vocab)
    x = randn(g, rows, vocab, dtype=DT[dt], scale=3.0)
    ids = torch.randint(0, vocab, (rows, 3), generator=g, device="cuda")
    r = check_logprobs(x, ids, top, temperature)
    for view in (strided(x, 1), strided(x, 7, 3)):  # rows that start anywhere
        v = check_logprobs(view, ids, top, temperature)
        if top:
            assert torch.equal(v.top_ids, r.top_ids)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [9000, 152064])
def test_logprobs_orders_that_overflow_the_candidates(vocab, dt):
    up = torch.linspace(-20, 20, vocab, device="cuda")
    rows = [up, up.flip(0), torch.zeros(vocab, device="cuda"), torch.where(torch.arange(vocab, device="cuda") % 2 == 0, -0.0, 0.0),
            torch.cat([torch.zeros(vocab - 2000, device="cuda"), torch.ones(2000, device="cuda")]),
            (torch.arange(vocab, device="cuda") % 777).float()]
    x = torch.stack(rows).to(DT[dt])
    ids = torch.tensor([[0, vocab - 1]] * len(rows), device="cuda")
    check_logprobs(x, ids, 64, 1.0)
    check_logprobs(x[:1], ids[:1], 5, 1.0)
    check_logprobs(x.repeat(80, 1), ids.repeat(80, 1), 20, 1.0)  # a CTA per row


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [6, 400])
def test_logprobs_masked_rows(rows, dt):
    vocab = 20000
    g = gen(5)
    x = randn(g, rows, vocab, dtype=DT[dt])
    lo = torch.finfo(DT[dt]).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 777] = 2.0
    x[2, 100:] = -math.inf
    x[3] = lo
    x[4] = lo
    x[4, 19999] = 1.0
    x[5, ::2] = lo
    ids = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
    ids[1, 0], ids[2, 0], ids[4, 0] = 777, 5, 19999
    r = check_logprobs(x, ids, 16, 1.0)
    assert r.top_ids[0].eq(-1).all() and r.entropy[0] == 0 and r.lse[0] == -math.inf
    assert r.top_ids[1, 0] == 777 and r.top_ids[1, 1] == -1 and r.logprobs[1, 0] == 0 and r.entropy[1] == 0


@pytest.mark.parametrize("rows", [3, 400])
def test_logprobs_nonfinite_rows_and_odd_ids(rows):
    x = randn(gen(6), rows, 5000)
    x[0, 3000] = math.nan
    x[1, 4000] = math.inf
    ids = torch.tensor([[-1, 0, 4999, 5000, 1 << 40]] * rows, device="cuda")
    r = ops.token_logprobs(x, ids, top=4)
    assert torch.isnan(r.entropy[:2]).all() and torch.isnan(r.lse[:2]).all()
    assert r.top_ids[:2].eq(-1).all() and torch.isnan(r.top_logprobs[:2]).all()
    assert torch.isnan(r.logprobs[:2, 1:]).all()
    assert r.logprobs[2:, 0].eq(0).all() and torch.isnan(r.logprobs[2:, 3:]).all()
    assert torch.isfinite(r.logprobs[2:, :3]).all() and torch.isfinite(r.entropy[2:]).all()
    one = ops.token_logprobs(x, ids[:, 1].contiguous())
    assert one.logprobs.shape == (rows,) and one.top_ids is None
    assert torch.equal(one.logprobs[2:], r.logprobs[2:, 1])


# ---------------------------------------------------------------------------
# Streams and graphs
# ---------------------------------------------------------------------------
def test_operators_run_on_the_current_stream_and_in_graphs():
    g = gen(11)
    x, h = randn(g, 20, 512, dtype=torch.bfloat16), randn(g, 20, 512)
    w, sw = ops.quantize_fp8_weight(randn(g, 1024, 512, scale=0.05))
    gain = 1 + randn(g, 512, scale=0.1)
    plan = ops.RotaryPlan(64)
    pos = torch.arange(20, device="cuda")

    def chain():
        r = ops.block_norm(x, h, post_gain=gain, pre_gain=gain, out_dtype=F8)
        o = ops.fp8_linear(r.out, r.scale, w, sw)
        q, _ = ops.rotary(o.view(20, 16, 64), None, pos, plan)
        lp = ops.token_logprobs(q.reshape(20, 1024), pos[:, None], top=3)
        return r.residual, o, q, lp.logprobs, lp.entropy, lp.top_ids

    want = [t.clone() for t in chain()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1000000)  # work queued before the inputs below are written
        x2 = x.clone()
        x.copy_(x2)
        got = chain()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ops.check_status()


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_refusals():
    x = torch.randn(4, 256, device="cuda", dtype=torch.bfloat16)
    q, s = ops.quantize_fp8(x)
    w, sw = ops.quantize_fp8_weight(x)
    plan = ops.RotaryPlan(64)
    heads = x.view(4, 4, 64)
    bad = [
        lambda: ops.quantize_fp8(x.cpu()),
        lambda: ops.quantize_fp8(x.double()),
        lambda: ops.quantize_fp8(x[0]),
        lambda: ops.quantize_fp8(x.T),
        lambda: ops.quantize_fp8(x, act="silu"),
        lambda: ops.quantize_fp8(x, gate=x, act="tanh"),
        lambda: ops.quantize_fp8(x, gate=x.float(), act="silu"),
        lambda: ops.quantize_fp8(x, gate=x[:2], act="silu"),
        lambda: ops.quantize_fp8(x.float().requires_grad_()),
        lambda: ops.fp8_linear(x, s, w, sw),
        lambda: ops.fp8_linear(q, s[:2], w, sw),
        lambda: ops.fp8_linear(q, s, w[:, :128], sw),
        lambda: ops.fp8_linear(q, s, w, sw.half()),
        lambda: ops.fp8_linear(q, s, w, sw, bias=torch.zeros(3, device="cuda")),
        lambda: ops.fp8_linear(q, s, w, sw, out_dtype=torch.float64),
        lambda: ops.fp8_linear(q, s, w, sw, out=torch.empty(4, 5, device="cuda", dtype=torch.bfloat16)),
        lambda: ops.block_norm(None, None),
        lambda: ops.block_norm(x, x.half()),
        lambda: ops.block_norm(x, x[:, :8]),
        lambda: ops.block_norm(x, x, post_gain=torch.ones(8, device="cuda")),
        lambda: ops.block_norm(x, x, post_gain=torch.ones(256, device="cuda", dtype=torch.bfloat16)),
        lambda: ops.block_norm(x, x, gate=torch.ones(3, 256, device="cuda")),
        lambda: ops.block_norm(x, x, out_dtype=F8),
        lambda: ops.block_norm(None, x, gate=x),
        lambda: ops.block_norm(x, None, in_place=True),
        lambda: ops.block_norm(torch.zeros(1, 16385, device="cuda"), None),
        lambda: ops.rotary(None, None, 0, plan),
        lambda: ops.rotary(heads, None, torch.zeros(3, device="cuda", dtype=torch.int64), plan),
        lambda: ops.rotary(heads, None, torch.zeros(4, device="cuda"), plan),
        lambda: ops.rotary(heads, heads.half(), 0, plan),
        lambda: ops.rotary(heads, heads[:2], 0, plan),
        lambda: ops.rotary(x.view(4, 2, 128), None, 0, plan),
        lambda: ops.RotaryPlan(64, rotary_dim=66),
        lambda: ops.RotaryPlan(64, rotary_dim=63),
        lambda: ops.RotaryPlan(64, layout="split"),
        lambda: ops.token_logprobs(x, top=65),
        lambda: ops.token_logprobs(x, torch.zeros(4, device="cuda", dtype=torch.int32)),
        lambda: ops.token_logprobs(x, torch.zeros(3, 1, device="cuda", dtype=torch.int64)),
        lambda: ops.token_logprobs(x.T),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was accepted")
    refused_by_the_library = [
        lambda: ops.fp8_linear(q.view(torch.uint8)[:, 1:129].view(F8), s[:, :1], w[:, :128], sw[:, :1]),
        lambda: ops.block_norm(x, x, residual_scale=math.inf),
        lambda: ops.block_norm(x, x, pre_gain=torch.ones(256, device="cuda"), eps=-1.0),
        lambda: ops.token_logprobs(x, temperature=0.0),
        lambda: ops.RotaryPlan(64, theta=-1.0),
        lambda: ops.RotaryPlan(64, scaling={"type": "yarn", "factor": 0.5, "original_max_position": 10}),
    ]
    for i, f in enumerate(refused_by_the_library):
        with pytest.raises(_abi.VdError):
            f()
            pytest.fail(f"case {i} was accepted")


# ---------------------------------------------------------------------------
# Rows far apart
# ---------------------------------------------------------------------------
def test_offsets_past_32_bits():
    """Rows 2^30 elements apart (the third starts past 2^31) give what the same rows give side by side."""
    step = 1 << 30
    buf = torch.empty(2 * step + 8192, dtype=torch.bfloat16, device="cuda")

    def far(t):
        v = buf.as_strided(t.shape, (step, 1))
        v.copy_(t)
        return v

    g = gen(21)
    x = randn(g, 3, 2056, dtype=torch.bfloat16, scale=2.0)
    gain = 1 + randn(g, 2056, scale=0.1)
    q, s = ops.quantize_fp8(x)
    qf, sf = ops.quantize_fp8(far(x))
    assert torch.equal(q.float(), qf.float()) and torch.equal(s, sf)
    r, rf = ops.block_norm(x, x, post_gain=gain, pre_gain=gain), ops.block_norm(far(x), x, post_gain=gain, pre_gain=gain)
    assert torch.equal(r.out, rf.out) and torch.equal(r.residual, rf.residual)
    ids = torch.tensor([[5, 2055]] * 3, device="cuda")
    lp, lpf = ops.token_logprobs(x, ids, top=7), ops.token_logprobs(far(x), ids, top=7)
    assert all(torch.equal(a, b) for a, b in zip(lp, lpf))
    w, sw = operand(g, 2056, 2056, 128)
    out = ops.fp8_linear(q, s, w, sw)
    assert torch.equal(ops.fp8_linear(q, s, w, sw, out=buf.as_strided((3, 2056), (step, 1))), out)
    a = buf.view(torch.uint8).as_strided((3, 2056), (step, 1))
    a.copy_(q.view(torch.uint8) if q.is_contiguous() else q.contiguous().view(torch.uint8))
    assert torch.equal(ops.fp8_linear(a.view(F8), s, w, sw), out)
    plan = ops.RotaryPlan(128)
    heads = x[:, :1024].unflatten(1, (8, 128))
    pos = torch.tensor([3, 70000, 1], device="cuda")
    want, _ = ops.rotary(heads, None, pos, plan)
    v = buf.as_strided((3, 8, 128), (step, 128, 1))
    v.copy_(heads)
    got, _ = ops.rotary(v, None, pos, plan, q_out=v)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_logprobs_bounds_that_rise_many_times(dt):
    """Rows of more than a hundred batches whose maxima keep rising: every doubling of what has been read raises the
    bound on the alternatives; the answer is the sorted one each time."""
    vocab = 1_050_000
    g = gen(31)
    ramp = torch.linspace(0, 6, vocab, device="cuda")
    x = (randn(g, 4, vocab) + ramp).to(DT[dt])
    x = x.repeat(150, 1) if dt == "bf16" else x.repeat(75, 1)
    ids = torch.zeros(x.shape[0], 1, dtype=torch.int64, device="cuda")
    first = check_logprobs(x[:4], ids[:4], 64, 1.0)
    for _ in range(5):
        r = ops.token_logprobs(x, ids, top=64)
        for i in range(0, x.shape[0], 4):
            assert torch.equal(r.top_ids[i:i + 4], first.top_ids)


@pytest.mark.parametrize("scaling", [
    None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
    {"type": "yarn", "factor": 4.0, "original_max_position": 4096},
    {"type": "llama3", "factor": 8.0, "original_max_position": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0}])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_far_positions_against_the_formula(scaling, inverse):
    """Frequencies from their formulas, not from the plan: a turn is off by at most 2^-62 per position."""
    from rotary_reference import fraction_of_a_turn, turns_per_position
    plan = ops.RotaryPlan(64, theta=1e6, scaling=scaling)
    pos = [1, 131071, (1 << 31) - 1, 1 << 33, (1 << 37) - 5, -(1 << 37), (1 << 45) + 12345]
    q = randn(gen(14), len(pos), 2, 64)
    out, _ = ops.rotary(q, None, torch.tensor(pos, device="cuda"), plan, inverse=inverse)
    turns = turns_per_position(64, 1e6, scaling)
    frac = [[fraction_of_a_turn(p, t) for t in turns] for p in pos]
    ang = 2 * math.pi * torch.tensor(frac, dtype=torch.float64, device="cuda")[:, None]
    c, s = ang.cos() * plan.factor, ang.sin() * plan.factor * (-1 if inverse else 1)
    a, b = q.double()[..., :32], q.double()[..., 32:]
    ref = torch.cat([a * c - b * s, b * c + a * s], -1)
    mag = torch.cat([a.abs() + b.abs()] * 2, -1)
    off = 2 * math.pi * torch.tensor(pos, dtype=torch.float64, device="cuda").abs()[:, None, None] * 2.0 ** -62
    within(out, ref, rotary_bound(ref, mag, plan, torch.float32) + off * plan.factor * mag)


def test_rotary_cosines_and_sines_near_quarter_turns():
    """Rotating (1, 0) gives the cosine and the sine themselves.  The turn is reduced before it is rounded, so each is
    right to a few units in its own last place, small ones beside a half or quarter turn too: 2^-24 for the rounded rest,
    one unit (at most 2^-23) for the function."""
    plan = ops.RotaryPlan(64, theta=1e4)
    pos = torch.randint(0, 131072, (4096,), generator=gen(41), device="cuda")
    q = torch.zeros(4096, 1, 64, device="cuda")
    q[..., :32] = 1
    out, _ = ops.rotary(q, None, pos, plan)
    mine = [t % (1 << 64) for t in plan.turns.tolist()]
    ang = 2 * math.pi * torch.tensor([[((p * t) % (1 << 64)) / 2.0 ** 64 for t in mine] for p in pos.tolist()],
                                     dtype=torch.float64, device="cuda")
    want = torch.cat([ang.cos(), ang.sin()], -1)[:, None]
    within(out, want, 4 * U * want.abs() + 1e-12)
    assert (want.abs() < 1e-4).sum() > 10  # some do lie there


def test_negated_views_are_refused():
    """Their memory holds the values with the other sign."""
    x = torch.randn(4, 256, device="cuda")
    neg = torch._neg_view(x)
    assert torch.equal(neg, -x) and neg.data_ptr() == x.data_ptr()
    for f in (lambda: ops.quantize_fp8(neg), lambda: ops.block_norm(neg, x), lambda: ops.token_logprobs(neg)):
        with pytest.raises(ValueError, match="resolve_neg"):
            f()
    assert torch.equal(ops.block_norm(neg.resolve_neg(), x).residual, torch.zeros_like(x))
