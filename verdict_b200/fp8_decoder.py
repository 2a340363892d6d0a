"""A decoder on 8-bit weights that scores answers: the operators of `ops.py` as they are used together.

    model = Fp8Decoder.synthetic(spec.preset("onejev-9b", layers=2))
    scored = model.score([(prompt_ids, answer_ids), ...], top=5)

Where the engine (`engine.py`) reads a decision from a handful of label rows,
this scores any answer: the log probability of each of its tokens over the whole
vocabulary, how uncertain the model was there (entropy, in nats) and what it
would rather have said.  One packed prefill over all pairs, per layer

    block_norm -> fp8_linear (q, k, v) -> rotary -> causal attention ->
    quantize_fp8 -> fp8_linear -> block_norm -> fp8_linear (gate, up) ->
    quantize_fp8 (act(gate) * up) -> fp8_linear

with the projections as e4m3 and a scale per block of 128, activations cast on
the way in, the residual stream in fp32, and the other activations in 16 bits.
Specs are the plain decoders of `spec.py` (styles "qwen3" and "gemma"), weights
a mapping by their Hugging Face names.  A spec may add "rope_scaling" (see
`ops.RotaryPlan`) and "post_norms": True with the weights
`post_self_attn_layernorm` and `post_mlp_layernorm` of each layer (a norm after
each block as well), "residual_scale" and "block_scale".

    python -m verdict_b200.fp8_decoder --preset onejev-9b --layers 2
"""

from __future__ import annotations

import argparse
import ctypes
import json
import math
from typing import Mapping, NamedTuple, Sequence, Tuple

import numpy as np
import torch

from . import _abi, ops
from . import spec as specs

DTYPE = torch.bfloat16


def _call(name: str, *args) -> None:
    err = ctypes.create_string_buffer(512)
    rc = getattr(_abi.load(), name)(*args, torch.cuda.current_stream().cuda_stream, err, len(err))
    _abi.check(rc, err)


class Scored(NamedTuple):
    logprob: float                 # of the whole answer
    token_logprobs: torch.Tensor   # [answer tokens]
    entropy: torch.Tensor          # [answer tokens]
    top_ids: torch.Tensor          # [answer tokens, top]
    top_logprobs: torch.Tensor


class _Projection(NamedTuple):
    q: torch.Tensor
    scale: torch.Tensor
    bias: torch.Tensor | None

    def __call__(self, x, x_scale):
        return ops.fp8_linear(x, x_scale, self.q, self.scale, bias=self.bias, out_dtype=DTYPE)


class Fp8Decoder:
    def __init__(self, spec: dict, weights: Mapping[str, torch.Tensor], device=None):
        if spec.get("arch") != "decoder" or spec.get("style") not in ("qwen3", "gemma"):
            raise ValueError("Fp8Decoder takes plain decoder specs (styles qwen3 and gemma)")
        if spec["head_dim"] not in (128, 256):
            raise ValueError("the attention kernel takes head_dim 128 or 256")
        self.spec = spec
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device or "cuda")
        if dev.type != "cuda":
            raise ValueError("Fp8Decoder runs on a CUDA device")
        if dev.index is None:  # the one that is current now, whichever is when it answers
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev

        def vector(name):
            return weights[name].to(dev, torch.float32).contiguous()

        def projection(*names, bias=False):
            q, scale = ops.quantize_fp8_weight(torch.cat([weights[n + ".weight"].to(dev, DTYPE) for n in names]))
            b = torch.cat([vector(n + ".bias") for n in names]) if bias else None
            return _Projection(q, scale, b)

        self.layers = []
        for i in range(spec["layers"]):
            p = f"model.layers.{i}."
            a = p + "self_attn."
            self.layers.append(dict(
                qkv=projection(a + "q_proj", a + "k_proj", a + "v_proj", bias=spec["qkv_bias"]),
                o=projection(a + "o_proj"),
                gate_up=projection(p + "mlp.gate_proj", p + "mlp.up_proj"),
                down=projection(p + "mlp.down_proj"),
                norm1=vector(p + "input_layernorm.weight"),
                norm2=vector(p + "post_attention_layernorm.weight"),
                q_norm=vector(a + "q_norm.weight") if spec["qk_norm"] else None,
                k_norm=vector(a + "k_norm.weight") if spec["qk_norm"] else None,
                post1=vector(p + "post_self_attn_layernorm.weight") if spec.get("post_norms") else None,
                post2=vector(p + "post_mlp_layernorm.weight") if spec.get("post_norms") else None,
            ))
        self.norm = vector("model.norm.weight")
        self.embed = weights["model.embed_tokens.weight"].to(dev, DTYPE)
        head = self.embed if spec["tied"] else weights["lm_head.weight"].to(dev, DTYPE)
        # The head's product takes rows in multiples of 128; the added ones are cut off its output.
        self.head = torch.nn.functional.pad(head, (0, 0, 0, -head.shape[0] % 128)).contiguous()
        self.rope = ops.RotaryPlan(spec["head_dim"], theta=spec["rope_theta"], scaling=spec.get("rope_scaling"),
                                   device=dev)

    @classmethod
    def synthetic(cls, spec: dict, seed: int = 0, device="cuda") -> "Fp8Decoder":
        """Random weights of the spec's shape (none ship with this package)."""
        return cls(spec, synthetic_weights(spec, seed, device))

    def _norm(self, y, h, post, pre, out_dtype):
        s = self.spec
        return ops.block_norm(y, h, post_gain=post, residual_scale=s.get("residual_scale", 1.0),
                              block_scale=s.get("block_scale", 1.0), pre_gain=pre, eps=s["rms_eps"],
                              plus_one=s["norm_plus_one"], out_dtype=out_dtype, in_place=True)

    def _attention(self, qkv, positions, lengths, layer):
        s = self.spec
        nq, nkv, hd = s["heads"], s["kv_heads"], s["head_dim"]
        tokens, width = qkv.shape
        q = qkv[:, :nq * hd].view(tokens, nq, hd)
        k = qkv[:, nq * hd:(nq + nkv) * hd].view(tokens, nkv, hd)
        if layer["q_norm"] is not None:
            def head_norm(x, gain):
                flat = x.reshape(-1, hd)
                return ops.block_norm(None, flat, pre_gain=gain, eps=s["rms_eps"],
                                      plus_one=s["norm_plus_one"]).out.view(x.shape)
            ops.rotary(head_norm(q, layer["q_norm"]), head_norm(k, layer["k_norm"]), positions, self.rope, q_out=q,
                       k_out=k)
        else:
            ops.rotary(q, k, positions, self.rope, q_out=q, k_out=k)
        out = torch.empty(tokens, nq * hd, dtype=DTYPE, device=qkv.device)
        cu = np.zeros(len(lengths) + 1, dtype=np.int32)
        np.cumsum(lengths, out=cu[1:])
        _call("vdk_attention_tc", qkv.data_ptr(), width, 0, nq * hd, (nq + nkv) * hd, nq, nkv, hd, _abi.VDK_BF16, 1,
              cu.ctypes.data, len(lengths), out.data_ptr(), nq * hd)
        return out

    @torch.no_grad()
    def hidden(self, ids: torch.Tensor, lengths: Sequence[int]) -> torch.Tensor:
        """Final normalised hidden states [tokens, hidden] of packed sequences: ids [tokens], their lengths."""
        s = self.spec
        with torch.cuda.device(self.device):
            h = self.embed[ids].float()
            if s["embed_scale"]:
                h *= math.sqrt(s["hidden"])
            positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in lengths]).to(self.device)
            f = s["ffn"]
            y, post = None, None
            for layer in self.layers:
                x = (self._norm(y, h, post, layer["norm1"], ops.FP8) if y is not None else
                     ops.block_norm(None, h, pre_gain=layer["norm1"], eps=s["rms_eps"], plus_one=s["norm_plus_one"],
                                    out_dtype=ops.FP8))
                attn = self._attention(layer["qkv"](x.out, x.scale), positions, lengths, layer)
                y = layer["o"](*ops.quantize_fp8(attn))
                x = self._norm(y, h, layer["post1"], layer["norm2"], ops.FP8)
                both = layer["gate_up"](x.out, x.scale)
                y = layer["down"](*ops.quantize_fp8(both[:, f:], gate=both[:, :f], act=s["act"]))
                post = layer["post2"]
            return self._norm(y, h, post, self.norm, DTYPE).out

    @torch.no_grad()
    def score(self, pairs: Sequence[Tuple[Sequence[int], Sequence[int]]], top: int = 5,
              temperature: float = 1.0) -> list:
        """One `Scored` per (prompt ids, answer ids); neither may be empty."""
        if not pairs:
            return []
        rows, targets, lengths, packed = [], [], [], []
        for prompt, answer in pairs:
            if len(prompt) == 0 or len(answer) == 0:
                raise ValueError("a prompt and an answer need at least one token each")
            start = len(packed)
            packed += list(prompt) + list(answer)
            # The token at position p is predicted by the hidden state at p - 1.
            rows += range(start + len(prompt) - 1, len(packed) - 1)
            targets += list(answer)
            lengths.append(len(prompt) + len(answer))
        if min(packed) < 0 or max(packed) >= self.embed.shape[0]:
            raise ValueError("a token id is outside the vocabulary")
        with torch.cuda.device(self.device):
            x = self.hidden(torch.tensor(packed, device=self.device), lengths)
            x = x[torch.tensor(rows, device=self.device)]
            n = self.head.shape[0]
            logits = torch.empty(x.shape[0], n, dtype=DTYPE, device=self.device)
            _call("vdk_gemm", x.data_ptr(), self.head.data_ptr(), x.shape[0], n, x.shape[1], _abi.VDK_BF16, 0, 0, None,
                  logits.data_ptr(), n)
            r = ops.token_logprobs(logits[:, :self.embed.shape[0]], torch.tensor(targets, device=self.device), top=top,
                                   temperature=temperature)
            ops.check_status(self.device)
        out, at = [], 0
        for _, answer in pairs:
            part = slice(at, at + len(answer))
            at += len(answer)
            lp = r.logprobs[part].cpu()
            out.append(Scored(float(lp.double().sum()), lp, r.entropy[part].cpu(),
                              r.top_ids[part].cpu() if top else None, r.top_logprobs[part].cpu() if top else None))
        return out


def synthetic_weights(spec: dict, seed: int = 0, device="cuda") -> dict:
    """Random weights by their Hugging Face names: normal with the spec's init_std, gains around one (zero where the
    norm adds one)."""
    g = torch.Generator(device=device).manual_seed(seed)
    d, f, hd = spec["hidden"], spec["ffn"], spec["head_dim"]
    base = 0.0 if spec["norm_plus_one"] else 1.0
    w = {}

    def matrix(name, rows, cols):
        w[name] = (torch.randn(rows, cols, generator=g, device=device) * spec["init_std"]).to(DTYPE)

    def gain(name, n):
        w[name] = base + 0.1 * torch.randn(n, generator=g, device=device)

    matrix("model.embed_tokens.weight", spec["vocab"], d)
    for i in range(spec["layers"]):
        p = f"model.layers.{i}."
        for n, rows, cols in (("q_proj", spec["heads"] * hd, d), ("k_proj", spec["kv_heads"] * hd, d),
                              ("v_proj", spec["kv_heads"] * hd, d), ("o_proj", d, spec["heads"] * hd)):
            matrix(f"{p}self_attn.{n}.weight", rows, cols)
            if spec["qkv_bias"] and n != "o_proj":
                w[f"{p}self_attn.{n}.bias"] = 0.02 * torch.randn(rows, generator=g, device=device)
        for n, rows, cols in (("gate_proj", f, d), ("up_proj", f, d), ("down_proj", d, f)):
            matrix(f"{p}mlp.{n}.weight", rows, cols)
        gain(p + "input_layernorm.weight", d)
        gain(p + "post_attention_layernorm.weight", d)
        if spec["qk_norm"]:
            gain(p + "self_attn.q_norm.weight", hd)
            gain(p + "self_attn.k_norm.weight", hd)
        if spec.get("post_norms"):
            gain(p + "post_self_attn_layernorm.weight", d)
            gain(p + "post_mlp_layernorm.weight", d)
    gain("model.norm.weight", d)
    if not spec["tied"]:
        matrix("lm_head.weight", spec["vocab"], d)
    return w


def main() -> None:
    ap = argparse.ArgumentParser(description="Score random answers with a synthetic decoder on 8-bit weights")
    ap.add_argument("--preset", default="onejev-9b", choices=["onejev-9b", "onejev-27b", "decider-2b"])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--pairs", type=int, default=8)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    spec = specs.preset(a.preset, layers=a.layers)
    model = Fp8Decoder.synthetic(spec, a.seed)
    rng = np.random.default_rng(a.seed)
    pairs = [(rng.integers(0, spec["vocab"], rng.integers(20, 600)).tolist(),
              rng.integers(0, spec["vocab"], rng.integers(1, 9)).tolist()) for _ in range(a.pairs)]
    for (prompt, answer), s in zip(pairs, model.score(pairs, top=3)):
        print(json.dumps(dict(prompt_tokens=len(prompt), answer=answer, logprob=round(s.logprob, 4),
                              entropy=[round(float(e), 4) for e in s.entropy], alternatives=s.top_ids.tolist())))


if __name__ == "__main__":
    main()
