"""Which outputs of the 8-bit decoder operators the C entries take: none that shares memory with another buffer."""

import ctypes
import os
import random
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import _abi, build, ops  # noqa: E402

PROGRAM = r"""
#include <cstdio>
#include "overlap.hpp"
int main() {
  long long v[12];
  while (true) {
    for (auto& x : v)
      if (std::scanf("%lld", &x) != 1) return 0;
    const vd::ByteRows a(reinterpret_cast<const void*>(v[0]), v[1], v[2], v[3], v[4], v[5]);
    const vd::ByteRows b(reinterpret_cast<const void*>(v[6]), v[7], v[8], v[9], v[10], v[11]);
    std::printf("%d %d\n", vd::overlap(a, b), vd::overlap(b, a));
  }
}
"""


def bytes_of(p, width, n0, s0, n1, s1):
    return {p + i * s0 + j * s1 + k for i in range(n0) for j in range(n1) for k in range(width)}


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_overlap_is_exact_where_the_outer_stride_is_shared(tmp_path):
    src, exe = tmp_path / "o.cpp", tmp_path / "o"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", build.CSRC, str(src), "-o", str(exe)], check=True)
    rng = random.Random(1)
    cases, want, exact = [], [], []
    for _ in range(20000):
        outer = rng.randint(6, 40)
        shared = rng.random() < 0.8

        def rows(base):
            width, n0, n1 = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 4)
            s1 = rng.choice([4, 5, 8, rng.randint(0, 12)])
            s0 = outer if shared else rng.randint(0, 60)
            if rng.random() < 0.5:
                n0, s0, n1, s1 = n1, s1, n0, s0
            return (base, width, n0, s0, n1, s1)
        a, b = rows(1000), rows(1000 + rng.randint(-60, 60))
        if a[0] == b[0] and rng.random() < 0.5:
            b = a
        cases.append(a + b)
        want.append(bool(bytes_of(*a) & bytes_of(*b)))

        def outers(r):
            # the stride the helper takes as the outer one, None where there is a single row
            live = [s for n, s in ((r[2], r[3]), (r[4], r[5])) if n > 1 and s > 0]
            return max(live) if live else None
        exact.append(outers(a) is None or outers(b) is None or outers(a) == outers(b))
    res = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases), text=True, capture_output=True,
                         check=True).stdout.split("\n")
    apart = 0
    for case, w, e, line in zip(cases, want, exact, res):
        ab, ba = (x == "1" for x in line.split())
        assert ab or not w, case       # never misses one
        assert ba or not w, case
        wide = any(s and s < width for width, n, s in ((case[1], case[2], case[3]), (case[1], case[4], case[5]),
                                                       (case[7], case[8], case[9]), (case[7], case[10], case[11])) if n > 1)
        if e and not wide:
            assert ab == w and ba == w, case
            apart += not w
    assert apart > 1000


def call(name, *args):
    err = ctypes.create_string_buffer(512)
    rc = getattr(_abi.load(), name)(*args, None, err, 512)
    return rc, err.value.decode()


def test_c_entries_refuse_outputs_that_share_memory():
    F = 1 << 20
    A, B, C, D, G, O, P, Q = (F + (i << 20) for i in range(8))
    quant = ["vdk_quantize_fp8", A, 128, B, 128, 4, 2, 128, 0, C, 128, D, 1]
    weight = ["vdk_quantize_fp8_weight", A, 128, 2, 128, 2, C, 128, D, 1]
    linear = ["vdk_fp8_linear", A, 128, B, 1, C, 128, D, 1, 4, 4, 128, G, O, 4, 0, P]
    norm = ["vdk_block_norm", A, 8, 0, B, 8, 2, C, D, 2, 8, 1, 1.0, 1.0, G, 1e-6, 0, 2, 8, O, 8, P, 8, 0, None, 0]
    norm8 = norm[:23] + [3, Q, 1]
    logp = ["vdk_token_logprobs", A, 20, 2, 20, 0, 1.0, B, 1, 3, C, D, G, O, P]
    # (entry, which argument, the address it gets): each inside another buffer
    for args, at, to in [
            (quant, 9, A), (quant, 9, B + 16), (quant, 11, A + 4), (quant, 11, C), (weight, 6, A), (weight, 8, C + 64),
            (linear, 13, A), (linear, 13, C + 16), (linear, 13, B), (linear, 13, D), (linear, 13, G + 8), (linear, 13, P),
            (norm, 19, A), (norm, 19, B + 4), (norm, 19, C), (norm, 19, D + 16), (norm, 19, G), (norm, 21, O),
            (norm, 21, A + 2), (norm, 21, B), (norm8, 21, A), (norm8, 21, Q), (norm8, 24, B), (norm8, 24, O + 4),
            (logp, 10, A), (logp, 11, B), (logp, 12, C), (logp, 13, G), (logp, 14, O)]:
        bad = list(args)
        bad[at] = to
        rc, msg = call(*bad)
        assert rc == _abi.VD_EINVAL and "overlap" in msg, (args[0], at, rc, msg)
    # A gate with one value a row, taken from the residual that is replaced in place.
    gate = list(norm)
    gate[4], gate[8], gate[10], gate[11], gate[19] = B, B, 8, 0, B
    rc, msg = call(*gate)
    assert rc == _abi.VD_EINVAL and "gate overlap" in msg, msg

    H = _abi.VdkRotaryHeads
    heads = lambda i, o: H(i, o, 128, 64, 128, 64, 2)  # noqa: E731  3 tokens, 2 heads of 64, fp16
    for q, k, pos, turns in [
            (heads(A, A + 128), heads(B, B), None, C), (heads(A, B), heads(B, C), None, D), (heads(A, A), heads(A, B), None, D),
            (heads(A, C), heads(B, C + 64), None, D), (heads(A, A), heads(A, A), None, D), (heads(A, B), None, B + 8, D),
            (heads(A, B), None, None, B + 8)]:
        rc, msg = call("vdk_rotary", q, k, 3, 64, 64, 0, 0, 0, pos, 64 if pos else 0, 0, turns, 1.0)
        assert rc == _abi.VD_EINVAL and "overlap" in msg, (rc, msg)


@pytest.mark.gpu
def test_views_of_one_packed_buffer_are_taken_and_shifted_ones_refused():
    plan = ops.RotaryPlan(64)
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(5, 6 * 64, generator=g, device="cuda")
    pos = torch.arange(5, device="cuda")
    # [q q q q | k | v] and heads of q, k and v in turn: rotated in place.
    for q, k in ((lambda t: t[:, :256].view(5, 4, 64), lambda t: t[:, 256:320].view(5, 1, 64)),
                 (lambda t: t.view(5, 2, 3, 64)[:, :, 0], lambda t: t.view(5, 2, 3, 64)[:, :, 1])):
        want = ops.rotary(q(base), k(base), pos, plan)
        buf = base.clone()
        ops.rotary(q(buf), k(buf), pos, plan, q_out=q(buf), k_out=k(buf))
        assert torch.equal(q(buf), want[0]) and torch.equal(k(buf), want[1])
        with pytest.raises(_abi.VdError, match="overlap"):
            ops.rotary(q(buf), None, pos, plan, q_out=buf.flatten()[32:].as_strided(q(buf).shape, q(buf).stride()))
        with pytest.raises(_abi.VdError, match="overlap"):
            ops.rotary(q(buf), q(buf), pos, plan, q_out=q(buf), k_out=q(buf))
    x = torch.randn(6, 256, generator=g, device="cuda")
    with pytest.raises(_abi.VdError, match="overlap"):
        ops.block_norm(x[1:].clone(), x[:5], gate=x[1:], in_place=True)
    with pytest.raises(_abi.VdError, match="overlap"):
        ops.block_norm(x[:5].clone(), x[:5], gate=x[:5, :1], in_place=True)
    # The residual itself as block output and gate: the same elements, read by the thread that writes them.
    y = x[:5].clone()
    want = y + y * y
    ops.block_norm(y, y, gate=y, in_place=True)
    assert torch.allclose(y, want, rtol=1e-6, atol=1e-6)
    q, s = ops.quantize_fp8(x)
    w, sw = ops.quantize_fp8_weight(x)
    with pytest.raises(_abi.VdError, match="overlap"):
        ops.fp8_linear(q, s, w, sw, out=q.view(torch.bfloat16)[:, :6])
