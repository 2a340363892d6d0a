"""The 8-bit decoder operators beside autograd: what has no derivative is refused, what is written is seen to be."""

import pytest

torch = pytest.importorskip("torch")

import torch.autograd.forward_ad as fwAD  # noqa: E402

from verdict_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu


def test_forward_mode_tangents_are_refused():
    x = torch.randn(4, 256, device="cuda")
    plan = ops.RotaryPlan(64)
    gain = torch.ones(256, device="cuda")
    q, s = ops.quantize_fp8(x)
    w, sw = ops.quantize_fp8_weight(x)
    bias = torch.zeros(4, device="cuda")
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        d = dual(x)
        assert not d.requires_grad
        for f in (lambda: ops.quantize_fp8(d), lambda: ops.quantize_fp8(x, gate=d, act="silu"),
                  lambda: ops.quantize_fp8_weight(d), lambda: ops.block_norm(d, x), lambda: ops.block_norm(x, d),
                  lambda: ops.block_norm(x, x, pre_gain=dual(gain)), lambda: ops.block_norm(x, x, gate=dual(gain)),
                  lambda: ops.rotary(d.view(4, 4, 64), None, 0, plan), lambda: ops.token_logprobs(d),
                  lambda: ops.fp8_linear(q, dual(s), w, sw), lambda: ops.fp8_linear(q, s, w, sw, bias=dual(bias))):
            with pytest.raises(ValueError, match="tangent"):
                f()
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # no_grad leaves forward mode on
            ops.quantize_fp8(d)
        ops.quantize_fp8(x)  # without a tangent
