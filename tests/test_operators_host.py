"""Host side of the 8-bit decoder operators: rotary frequencies, argument checks of the C entries, refusals without a GPU."""

import ctypes
import math
from decimal import Decimal

import pytest

torch = pytest.importorskip("torch")

from rotary_reference import fraction_of_a_turn, turns_per_position  # noqa: E402
from verdict_b200 import _abi, ops  # noqa: E402


def radians(turns):
    return [2 * math.pi * t / 2.0 ** 64 for t in turns]


def plain(rd, theta):
    return [theta ** (-2.0 * i / rd) for i in range(rd // 2)]


def close(got, want):
    for g, w in zip(got, want):
        # whole turns drop out; a double's 53 bits on a frequency of at most one radian
        assert abs(math.remainder(g - w, 2 * math.pi)) <= 2.0 ** -50, (g, w)


def test_rotary_turns_plain_and_linear():
    for rd, theta in ((2, 1e4), (64, 1e4), (128, 1e6)):
        t, m = ops.rotary_turns(rd, theta)
        assert m == 1.0 and len(t) == rd // 2
        close(radians(t), plain(rd, theta))
        t, m = ops.rotary_turns(rd, theta, {"type": "linear", "factor": 4.0})
        close(radians(t), [f / 4 for f in plain(rd, theta)])


def test_rotary_turns_ntk():
    t, _ = ops.rotary_turns(64, 1e4, {"type": "ntk", "factor": 8.0})
    close(radians(t), plain(64, 1e4 * 8.0 ** (64 / 62)))
    # The slowest pair ends up divided by the factor, the fastest as it was.
    close(radians(t)[-1:], [plain(64, 1e4)[-1] / 8])


def test_rotary_turns_yarn_matches_a_worked_ramp():
    rd, theta, orig, factor = 128, 1e6, 32768, 4.0
    t, m = ops.rotary_turns(rd, theta, {"type": "yarn", "factor": factor, "original_max_position": orig})
    assert m == pytest.approx(0.1 * math.log(4) + 1, rel=1e-7)
    f = plain(rd, theta)
    turns_in_context = [x * orig / (2 * math.pi) for x in f]
    got = radians(t)
    for i in range(rd // 2):
        if turns_in_context[i] > 40:
            close([got[i]], [f[i]])
        elif turns_in_context[i] < 0.9:
            close([got[i]], [f[i] / factor])
        else:
            assert f[i] / factor * (1 - 1e-12) <= got[i] <= f[i] * (1 + 1e-12)
    assert all(a >= b for a, b in zip(got, got[1:]))
    _, m = ops.rotary_turns(rd, theta, {"type": "yarn", "factor": 4.0, "original_max_position": orig,
                                        "attention_factor": 1.25})
    assert m == 1.25


def test_rotary_turns_llama3_bands():
    rd, theta, orig, factor = 128, 5e5, 8192, 8.0
    t, m = ops.rotary_turns(rd, theta, {"type": "llama3", "factor": factor, "original_max_position": orig,
                                        "low_freq_factor": 1.0, "high_freq_factor": 4.0})
    assert m == 1.0
    for got, f in zip(radians(t), plain(rd, theta)):
        wave = 2 * math.pi / f
        if wave < orig / 4:
            want = f
        elif wave > orig:
            want = f / factor
        else:
            s = (orig / wave - 1) / 3
            want = (1 - s) * f / factor + s * f
        close([got], [want])


def test_rotary_turns_divisors():
    d = [1.0 + i for i in range(8)]
    t, m = ops.rotary_turns(16, 1e4, {"type": "divisors", "divisors": d, "attention_factor": 1.5})
    assert m == 1.5
    close(radians(t), [f / x for f, x in zip(plain(16, 1e4), d)])


@pytest.mark.parametrize("rd,scaling", [
    (3, None), (0, None), (2048, None), (64, {"type": "cubic"}), (64, {"type": "linear"}),
    (64, {"type": "linear", "factor": 2.0, "extra": 1}), (64, {"type": "divisors", "divisors": [1.0]})])
def test_rotary_turns_refusals(rd, scaling):
    with pytest.raises(ValueError):
        ops.rotary_turns(rd, 1e4, scaling)


@pytest.mark.parametrize("theta,scaling", [
    (0.0, None), (math.nan, None), (1e4, {"type": "linear", "factor": 0.5}),
    (1e4, {"type": "yarn", "factor": 2.0, "original_max_position": 0}),
    (1e4, {"type": "llama3", "factor": 2.0, "original_max_position": 8, "low_freq_factor": 4.0, "high_freq_factor": 1.0}),
    (1e4, {"type": "divisors", "divisors": [0.0] * 32})])
def test_rotary_turns_values_refused_by_the_library(theta, scaling):
    with pytest.raises(_abi.VdError) as e:
        ops.rotary_turns(64, theta, scaling)
    assert e.value.code == _abi.VD_EINVAL


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 128)
    for f in (lambda: ops.quantize_fp8(x), lambda: ops.quantize_fp8_weight(x), lambda: ops.block_norm(x, x),
              lambda: ops.token_logprobs(x), lambda: ops.quantize_fp8("x")):
        with pytest.raises(ValueError):
            f()


def call(name, *args):
    err = ctypes.create_string_buffer(512)
    rc = getattr(_abi.load(), name)(*args, None, err, 512)
    return rc, err.value.decode()


FAKE = 1 << 20  # an address that no check reads


def test_c_entries_check_before_they_launch():
    """Bad arguments come back as VD_EINVAL with a message; zero rows are no work.  No device is needed for either."""
    E = _abi.VD_EINVAL
    cases = [
        ("vdk_quantize_fp8", (FAKE, 128, None, 0, 0, -1, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8", (FAKE, 100, None, 0, 0, 2, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8", (FAKE, 128, None, 0, 4, 2, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8", (None, 128, None, 0, 0, 2, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8", (FAKE, 128, None, 0, 0, 2, 128, 7, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8", (FAKE, 128, None, 0, 0, 1 << 40, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8_weight", (FAKE, 128, 0, 128, 0, FAKE, 128, FAKE, 1)),
        ("vdk_quantize_fp8_weight", (FAKE, 128, 4, 128, 9, FAKE, 128, FAKE, 1)),
        ("vdk_fp8_linear", (FAKE, 128, FAKE, 1, FAKE, 128, FAKE, 1, 4, 4, 0, None, FAKE, 4, 0, None)),
        ("vdk_fp8_linear", (FAKE + 8, 128, FAKE, 1, FAKE, 128, FAKE, 1, 4, 4, 128, None, FAKE, 4, 0, None)),
        ("vdk_fp8_linear", (FAKE, 136, FAKE, 1, FAKE, 128, FAKE, 1, 4, 4, 128, None, FAKE, 4, 0, None)),
        ("vdk_fp8_linear", (FAKE, 128, FAKE, 0, FAKE, 128, FAKE, 1, 4, 4, 128, None, FAKE, 4, 0, None)),
        ("vdk_fp8_linear", (FAKE, 128, FAKE, 1, FAKE, 128, FAKE, 1, 4, 4, 128, None, FAKE, 3, 0, None)),
        ("vdk_fp8_linear", (FAKE, 128, FAKE, 1, FAKE, 128, FAKE, 1, 4, 4, 128, None, FAKE, 4, 3, None)),
        ("vdk_block_norm", (FAKE, 8, 0, FAKE, 8, 1, None, None, 0, 0, 0, 1.0, 1.0, None, 1e-6, 0, 2, 8, FAKE, 8, None, 0,
                            0, None, 0)),
        ("vdk_block_norm", (FAKE, 8, 0, FAKE, 8, 2, None, None, 0, 0, 0, 1.0, 1.0, None, 1e-6, 0, 2, 8, None, 8, None, 0,
                            0, None, 0)),
        ("vdk_block_norm", (FAKE, 8, 0, FAKE, 8, 2, None, FAKE, 2, 8, 2, 1.0, 1.0, None, 1e-6, 0, 2, 8, FAKE, 8, None, 0,
                            0, None, 0)),
        ("vdk_block_norm", (FAKE, 8, 0, FAKE, 8, 2, None, None, 0, 0, 0, 1.0, 1.0, FAKE, 1e-6, 0, 2, 8, FAKE, 8, FAKE, 8,
                            3, None, 0)),
        ("vdk_block_norm", (FAKE, 20000, 0, None, 0, 2, None, None, 0, 0, 0, 1.0, 1.0, None, 1e-6, 0, 2, 20000, FAKE,
                            20000, None, 0, 0, None, 0)),
        ("vdk_rotary", (None, None, 2, 64, 64, 0, 0, 0, None, 0, 0, FAKE, 1.0)),
        ("vdk_rotary", (_abi.VdkRotaryHeads(FAKE, FAKE, 64, 64, 64, 0, 2), None, 2, 64, 64, 0, 0, 0, None, 0, 0, FAKE, 1.0)),
        ("vdk_rotary", (_abi.VdkRotaryHeads(FAKE, FAKE, 64, 64, 64, 64, 1), None, 2, 64, 65, 0, 0, 0, None, 0, 0, FAKE, 1.0)),
        ("vdk_rotary", (_abi.VdkRotaryHeads(FAKE, FAKE, 64, 64, 64, 64, 1), None, 2, 64, 64, 0, 0, 0, FAKE, 16, 0, FAKE, 1.0)),
        ("vdk_rotary", (_abi.VdkRotaryHeads(FAKE, FAKE, 64, 64, 64, 64, 1), None, 2, 64, 64, 0, 0, 0, None, 0, 0, None, 1.0)),
        ("vdk_token_logprobs", (FAKE, 10, 2, 20, 0, 1.0, None, 0, 0, None, None, None, None, None)),
        ("vdk_token_logprobs", (FAKE, 20, 2, 20, 0, 0.0, None, 0, 0, None, None, None, None, None)),
        ("vdk_token_logprobs", (FAKE, 20, 2, 20, 0, 1.0, None, 0, 65, None, None, None, FAKE, FAKE)),
        ("vdk_token_logprobs", (FAKE, 20, 2, 20, 0, 1.0, None, 2, 0, FAKE, None, None, None, None)),
        ("vdk_token_logprobs", (FAKE, 20, 2, 20, 0, 1.0, None, 0, 3, None, None, None, None, FAKE)),
    ]
    for name, args in cases:
        rc, msg = call(name, *args)
        assert rc == E and msg, (name, args, rc, msg)
    nothing = [
        ("vdk_quantize_fp8", (None, 128, None, 0, 0, 0, 128, 0, None, 128, None, 1)),
        ("vdk_fp8_linear", (None, 128, None, 1, FAKE, 128, FAKE, 1, 0, 4, 128, None, None, 4, 0, None)),
        ("vdk_block_norm", (None, 8, 0, None, 8, 2, None, None, 0, 0, 0, 1.0, 1.0, None, 1e-6, 0, 0, 8, None, 8, None, 0,
                            0, None, 0)),
        ("vdk_token_logprobs", (None, 20, 0, 20, 0, 1.0, None, 0, 0, None, None, None, None, None)),
    ]
    for name, args in nothing:
        assert call(name, *args)[0] == _abi.VD_OK, name
    # A null error buffer is allowed.
    assert _abi.load().vdk_token_logprobs(FAKE, 10, 2, 20, 0, 1.0, None, 0, 0, None, None, None, None, None, None, None,
                                          0) == E


def test_rotary_outputs_that_overlap_are_refused():
    H = _abi.VdkRotaryHeads
    # (token stride, head stride) of 3 tokens x 2 heads of 64
    for token, head in ((64, 64), (0, 64), (100, 64), (64, 100), (32, 128)):
        rc, msg = call("vdk_rotary", H(FAKE, FAKE, 128, 64, token, head, 2), None, 3, 64, 64, 0, 0, 0, None, 0, 0, FAKE,
                       1.0)
        assert rc == _abi.VD_EINVAL and "overlap" in msg, (token, head, msg)


def test_limits_of_the_failure_path_entry():
    # zero rows: nothing is launched, only the limits are looked at
    args = (None, 128, None, 1, FAKE, 128, FAKE, 1, 0, 4, 128, None, None, 4, 0, None)
    assert call("vdk_fp8_linear_stalled", *args, 1000, -1)[0] == _abi.VD_OK
    for limit, stall in ((0, 0), (-1, 0), (2000001, 0), (1000, -2)):
        rc, msg = call("vdk_fp8_linear_stalled", *args, limit, stall)
        assert rc == _abi.VD_EINVAL and msg


def test_c_entries_refuse_pointers_off_their_element():
    """A kernel would fault on them; every pointer that one dereferences is looked at before a launch."""
    F, H = FAKE, _abi.VdkRotaryHeads
    # Far apart, so that nothing overlaps.
    A, B, C, D, G, O = (F + (i << 20) for i in range(6))
    quant = ["vdk_quantize_fp8", A, 128, B, 128, 4, 2, 128, 0, C, 128, D, 1]
    weight = ["vdk_quantize_fp8_weight", A, 128, 2, 128, 2, C, 128, D, 1]
    linear = ["vdk_fp8_linear", A, 128, B, 1, C, 128, D, 1, 4, 4, 128, G, O, 4, 0, F - 64]
    norm = ["vdk_block_norm", A, 8, 0, B, 8, 2, C, D, 2, 8, 1, 1.0, 1.0, G, 1e-6, 0, 2, 8, O, 8, O + (1 << 20), 8, 0, None,
            0]
    norm8 = norm[:23] + [3, F - 64, 1]
    logp = ["vdk_token_logprobs", A, 20, 2, 20, 0, 1.0, B, 1, 3, C, D, G, O, O + (1 << 20)]
    cases = [(quant, 1, 1), (quant, 3, 1), (quant, 11, 2), (weight, 1, 2), (weight, 8, 1), (linear, 3, 2), (linear, 7, 2),
             (linear, 12, 2), (linear, 13, 1), (linear, 16, 2), (norm, 1, 1), (norm, 4, 2), (norm, 7, 2), (norm, 8, 2),
             (norm, 14, 2), (norm, 19, 2), (norm, 21, 1), (norm8, 24, 2), (logp, 1, 1), (logp, 7, 4), (logp, 10, 2),
             (logp, 11, 2), (logp, 12, 2), (logp, 13, 2), (logp, 14, 2)]
    for args, at, off in cases:
        bad = list(args)
        assert isinstance(bad[at], int) and bad[at] >= F - 64, (args, at)
        bad[at] += off
        rc, msg = call(*bad)
        assert rc == _abi.VD_EINVAL and "aligned" in msg, (args[0], at, rc, msg)
    for heads, pos, bits, turns in ((H(A + 1, B, 128, 64, 128, 64, 2), None, 0, C), (H(A, B + 1, 128, 64, 128, 64, 2), None, 0, C),
                                    (H(A, B, 128, 64, 128, 64, 2), D + 2, 32, C), (H(A, B, 128, 64, 128, 64, 2), D + 4, 64, C),
                                    (H(A, B, 128, 64, 128, 64, 2), None, 0, C + 4)):
        rc, msg = call("vdk_rotary", heads, None, 3, 64, 64, 0, 0, 0, pos, bits, 0, turns, 1.0)
        assert rc == _abi.VD_EINVAL and "aligned" in msg, msg


def test_quantize_row_count_does_not_wrap():
    # rows * blocks is 4 modulo 2^64
    rc, msg = call("vdk_quantize_fp8", FAKE, 512, None, 0, 0, (1 << 62) + 1, 512, 0, 2 * FAKE, 512, 3 * FAKE, 4)
    assert rc == _abi.VD_EINVAL and "2^31" in msg


SCALINGS = [
    None, {"type": "linear", "factor": 3.0}, {"type": "ntk", "factor": 8.0},
    {"type": "yarn", "factor": 4.0, "original_max_position": 4096},
    {"type": "llama3", "factor": 8.0, "original_max_position": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
    {"type": "divisors", "divisors": [1.0 + i / 7 for i in range(48)]}]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("rd,theta", [(96, 1e4), (96, 1e6), (96, 5e5)])
def test_rotary_turns_have_all_their_64_bits(rd, theta, scaling):
    """Against 70 digits.  In units of 2^-64 of a turn, at up to 0.16 turns: half a unit for the rounding, and a long
    double's 2^-64 relative (0.16 units) for each of at most ten operations on the way (the power counts for two)."""
    turns, _ = ops.rotary_turns(rd, theta, scaling)
    for got, want in zip(turns, turns_per_position(rd, theta, scaling)):
        off = fraction_of_a_turn(1, Decimal(got) / 2 ** 64 - want) * 2.0 ** 64
        assert abs(off) <= 4, off


def test_logprobs_temperature_whose_exponent_factor_overflows_is_refused():
    # 1 / temperature is an fp32 number, log2(e) / temperature is not
    for t in (3.0e-39, 4.2e-39):
        rc, msg = call("vdk_token_logprobs", FAKE, 20, 2, 20, 0, t, None, 0, 0, None, None, None, None, None)
        assert rc == _abi.VD_EINVAL and "temperature" in msg, (t, rc, msg)


def test_a_products_plan_checks_its_arguments():
    for args in ((4, 4, 128, 3, FAKE, FAKE, FAKE), (0, 4, 128, 0, FAKE, FAKE, FAKE), (4, 4, 128, 0, None, FAKE, FAKE)):
        err = ctypes.create_string_buffer(512)
        assert _abi.load().vdk_fp8_linear_plan(*args, err, 512) == _abi.VD_EINVAL and err.value
