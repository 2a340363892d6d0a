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


def test_writes_count_in_the_tensors_version():
    x = torch.randn(4, 256, device="cuda")
    q, s = ops.quantize_fp8(x)
    w, sw = ops.quantize_fp8_weight(x)
    out = torch.empty(4, 4, device="cuda", dtype=torch.bfloat16)
    h, heads, ko = x.clone(), x.clone().view(4, 4, 64), torch.empty(4, 4, 64, device="cuda")
    before = [t._version for t in (out, h, heads, ko, x, q)]
    ops.fp8_linear(q, s, w, sw, out=out)
    ops.block_norm(x, h, in_place=True)
    ops.rotary(heads, x.view(4, 4, 64), 0, ops.RotaryPlan(64), q_out=heads, k_out=ko)
    after = [t._version for t in (out, h, heads, ko, x, q)]
    assert [a - b for a, b in zip(after, before)] == [1, 1, 1, 1, 0, 0]
    # So a tensor that autograd saved is missed when it is overwritten.
    leaf = torch.ones(4, 256, device="cuda", requires_grad=True)
    saved = torch.randn(4, 256, device="cuda")
    product = (leaf * saved).sum()
    ops.block_norm(x, saved, in_place=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    # Nothing is written: a residual that is handed through, no rows.
    b = h._version
    ops.block_norm(None, h, pre_gain=torch.ones(256, device="cuda"), in_place=True)
    ops.block_norm(x[:0], h[:0], in_place=True)
    assert h._version == b
    with torch.inference_mode():
        i = torch.zeros(4, 256, device="cuda")
    ops.block_norm(x, i, in_place=True)
    assert torch.equal(i, x)
