"""The 8-bit decoder (verdict_b200/fp8_decoder.py) against the same layers in 64 bits.

The reference rounds where the model stores: activations to 16 bits, casts to 8
bits, everything between in 64 bits.  Its attention is the library's kernel on
the reference's own q, k and v (tests/test_kernels_gpu.py holds that kernel to
its reference): that one keeps softmax weights in 16 bits, scaled to a running
maximum, and the next cast would turn that difference into whole steps.  The GPU's own fp32 arithmetic can still
put a value that lies near a rounding boundary on its other side, which moves
it by one step of the format; the cast itself moves every value by up to half
a step.  So the GPU's deviation from the reference has to stay below half of
what the casts do to the result (reference with casts against reference
without).
"""

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import _abi  # noqa: E402
from verdict_b200 import spec as specs  # noqa: E402

pytestmark = pytest.mark.gpu


def f8(c, amax):
    """The cast's definition, in fp32: 16-bit weights often lie on a rounding boundary exactly."""
    c, a = c.float(), amax.float().clamp_min(1e-30)
    limit = torch.full_like(a, 448.0)
    return (c * (limit / a)).to(torch.float8_e4m3fn).double() * (a / limit).double()


def cast(x):
    return torch.cat([f8(c, c.abs().amax(1, keepdim=True)) for c in x.split(128, 1)], 1)


def cast_weight(w):
    rows = []
    for r in w.split(128, 0):
        rows.append(torch.cat([f8(c, c.abs().max()) for c in r.split(128, 1)], 1))
    return torch.cat(rows, 0)


def rms(x, gain, spec):
    return x / (x.pow(2).mean(-1, keepdim=True) + spec["rms_eps"]).sqrt() * (gain + (1 if spec["norm_plus_one"] else 0))


def r16(x):
    return x.to(torch.bfloat16).double()


def attention(qkv, nq, nkv, hd):
    out = torch.empty(qkv.shape[0], nq * hd, dtype=qkv.dtype, device="cuda")
    cu = np.array([0, qkv.shape[0]], dtype=np.int32)
    err = ctypes.create_string_buffer(512)
    rc = _abi.load().vdk_attention_tc(qkv.data_ptr(), qkv.shape[1], 0, nq * hd, (nq + nkv) * hd, nq, nkv, hd,
                                      _abi.VDK_BF16, 1, cu.ctypes.data, 1, out.data_ptr(), nq * hd, None, err, len(err))
    _abi.check(rc, err)
    return out.double()


def reference_hidden(spec, weights, ids, lengths, casts):
    q8 = cast if casts else (lambda t: t)
    w8 = cast_weight if casts else (lambda t: t)
    W = {k: v.double() for k, v in weights.items()}
    nq, nkv, hd = spec["heads"], spec["kv_heads"], spec["head_dim"]
    rs, bs = spec.get("residual_scale", 1.0), spec.get("block_scale", 1.0)
    act = {"silu": torch.nn.functional.silu,
           "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[spec["act"]]
    outs = []
    inv = spec["rope_theta"] ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    if spec.get("rope_scaling"):
        inv = inv / spec["rope_scaling"]["factor"]
    start = 0
    for n in lengths:
        h = W["model.embed_tokens.weight"][ids[start:start + n]]
        start += n
        if spec["embed_scale"]:
            h = h * math.sqrt(spec["hidden"])
        ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None, None] * inv
        cos, sin = ang.cos(), ang.sin()

        def rot(x):
            a, b = x[..., :hd // 2], x[..., hd // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        for i in range(spec["layers"]):
            p = f"model.layers.{i}."

            def lin(x, name):
                y = q8(x) @ w8(W[p + name + ".weight"]).T
                return r16(y + W[p + name + ".bias"] if p + name + ".bias" in W else y)

            x = rms(h, W[p + "input_layernorm.weight"], spec)
            q = lin(x, "self_attn.q_proj").view(n, nq, hd)
            k = lin(x, "self_attn.k_proj").view(n, nkv, hd)
            v = lin(x, "self_attn.v_proj").view(n, nkv, hd)
            if spec["qk_norm"]:
                q = r16(rms(q, W[p + "self_attn.q_norm.weight"], spec))
                k = r16(rms(k, W[p + "self_attn.k_norm.weight"], spec))
            qkv = torch.cat([rot(q).flatten(1), rot(k).flatten(1), v.flatten(1)], 1).to(torch.bfloat16)
            y = lin(attention(qkv, nq, nkv, hd), "self_attn.o_proj")
            if spec.get("post_norms"):
                y = rms(y, W[p + "post_self_attn_layernorm.weight"], spec)
            h = rs * h + bs * y
            x = rms(h, W[p + "post_attention_layernorm.weight"], spec)
            y = lin(act(lin(x, "mlp.gate_proj")) * lin(x, "mlp.up_proj"), "mlp.down_proj")
            if spec.get("post_norms"):
                y = rms(y, W[p + "post_mlp_layernorm.weight"], spec)
            h = rs * h + bs * y
        outs.append(rms(h, W["model.norm.weight"], spec))
    return torch.cat(outs)


CASES = {
    "qwen3": dict(preset="onejev-9b", hidden=512, heads=4, kv_heads=2, ffn=1152, vocab=1000, init_std=0.05),
    "qwen2-bias": dict(preset="onejev-9b", hidden=384, heads=3, kv_heads=1, ffn=640, vocab=999, qk_norm=False,
                       qkv_bias=True, init_std=0.05, rope_scaling={"type": "linear", "factor": 2.0}),
    "gemma": dict(preset="decider-2b", hidden=512, heads=2, kv_heads=1, ffn=1024, vocab=1280, init_std=0.05),
    "both-norms": dict(preset="onejev-9b", hidden=512, heads=4, kv_heads=2, ffn=1024, vocab=1000, init_std=0.05,
                       post_norms=True, residual_scale=0.9, block_scale=0.5),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_scores_follow_the_64_bit_layers(name):
    from verdict_b200.fp8_decoder import Fp8Decoder, synthetic_weights
    kw = dict(CASES[name])
    spec = specs.preset(kw.pop("preset"), layers=2, **kw)
    weights = synthetic_weights(spec, 7)
    model = Fp8Decoder(spec, weights)
    g = torch.Generator().manual_seed(3)
    lengths = [(1, 1), (5, 3), (130, 7), (64, 1), (300, 20)]
    pairs = [(torch.randint(0, spec["vocab"], (a,), generator=g).tolist(),
              torch.randint(0, spec["vocab"], (b,), generator=g).tolist()) for a, b in lengths]
    ids = torch.tensor([t for p, a in pairs for t in p + a], device="cuda")
    lens = [a + b for a, b in lengths]
    got = model.hidden(ids, lens).double()
    with_casts = reference_hidden(spec, weights, ids, lens, True)
    without = reference_hidden(spec, weights, ids, lens, False)
    off, casts = (got - with_casts).norm(), (with_casts - without).norm()
    assert off <= 0.5 * casts, (float(off), float(casts))

    # The readout on top, from the GPU's own hidden states: 16-bit logits (relative 2^-8 of each).
    scored = model.score(pairs, top=4)
    head = weights["model.embed_tokens.weight"] if spec["tied"] else weights["lm_head.weight"]
    start = 0
    for (prompt, answer), s in zip(pairs, scored):
        rows = got[start + len(prompt) - 1:start + len(prompt) + len(answer) - 1]
        start += len(prompt) + len(answer)
        z = rows @ head.double().T
        lp = torch.log_softmax(z, 1)
        want = lp.gather(1, torch.tensor(answer, device="cuda")[:, None])[:, 0].cpu()
        slack = 2 * 2.0 ** -8 * float(z.abs().max()) + 1e-3
        assert (s.token_logprobs.double() - want).abs().max() <= slack
        assert abs(s.logprob - float(s.token_logprobs.double().sum())) < 1e-6
        assert s.top_ids.shape == (len(answer), 4) and (s.top_logprobs[:, 0] >= s.token_logprobs - 1e-6).all()
        best = lp.max(1).values.cpu()
        assert (s.top_logprobs[:, 0].double() - best).abs().max() <= slack


def test_refusals_and_empty_input():
    from verdict_b200.fp8_decoder import Fp8Decoder
    kw = dict(CASES["qwen3"])
    model = Fp8Decoder.synthetic(specs.preset(kw.pop("preset"), layers=1, **kw))
    assert model.score([]) == []
    for pairs in ([([], [1])], [([1], [])], [([1], [1000])], [([-1], [1])]):
        with pytest.raises(ValueError):
            model.score(pairs)
    with pytest.raises(ValueError):
        Fp8Decoder(specs.preset("laya-bert"), {})
    with pytest.raises(ValueError):
        Fp8Decoder(specs.preset("onejev16-9b"), {})


def test_the_model_stays_on_the_device_it_was_built_on():
    from verdict_b200.fp8_decoder import Fp8Decoder, synthetic_weights
    kw = dict(CASES["qwen3"])
    spec = specs.preset(kw.pop("preset"), layers=1, **kw)
    here = torch.cuda.current_device()
    for device in (None, "cuda", torch.device("cuda"), here, f"cuda:{here}"):
        model = Fp8Decoder(spec, synthetic_weights(spec), device=device)
        assert model.device == torch.device("cuda", here) == model.embed.device, device
    with pytest.raises(ValueError):
        Fp8Decoder(spec, {}, device="cpu")
