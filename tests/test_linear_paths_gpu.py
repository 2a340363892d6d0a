"""fp8_linear's few-rows kernel along its long paths, against the definition in 64 bits.

Short products hand a CTA one chunk of scales and less than one turn of its
ring of stages.  Here each CTA goes through several of both, in every width of
tile, and with the shallow ring that two CTAs on an SM have; how each shape is
run is asked for and asserted, so that another rule cannot leave these paths
out unseen.
"""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_operators_gpu import DT, gen, linear_bound, linear_ref, operand, randn, within  # noqa: E402
from verdict_b200 import _abi, ops  # noqa: E402

pytestmark = pytest.mark.gpu

SCALE_BLOCKS = {16: 16, 32: 16, 64: 8, 128: 8}   # k-blocks of scales in a chunk
DEEP = {16: 8, 32: 8, 64: 6, 128: 4}             # stages of a CTA that has its SM to itself


def plan(m, n, k, dtype=_abi.VDK_BF16):
    out = [ctypes.c_int(-1) for _ in range(3)]
    err = ctypes.create_string_buffer(512)
    _abi.check(_abi.load().vdk_fp8_linear_plan(m, n, k, dtype, *(ctypes.byref(x) for x in out), err, 512), err)
    return tuple(x.value for x in out)


# (shape, tile, whether K is shared, whether two CTAs share an SM)
CASES = [
    ((1, 256, 16384), 16, True, False), ((7, 130, 16500), 16, True, False), ((16, 24576, 4096), 16, False, True),
    ((13, 20001, 4200), 16, False, True),
    ((20, 300, 20000), 32, True, False), ((32, 256, 32768), 32, True, False), ((32, 24576, 4100), 32, False, True),
    ((37, 4096, 12288), 64, True, None), ((64, 300, 20000), 64, True, False), ((50, 20000, 1100), 64, False, True),
    ((64, 24576, 4096), 64, False, True),
    ((100, 4096, 12288), 128, True, False), ((128, 1000, 9000), 128, True, False), ((128, 1000, 10000), 128, True, False),
    ((200, 4096, 4096), 128, True, False),
]
ONE_CHUNK = [(128, 1000, 9000)]  # a share of K of 8 blocks: the ring alone turns


@pytest.mark.parametrize("shape,tile,shared,two", CASES)
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_several_chunks_and_turns_of_the_ring(shape, tile, shared, two, dt):
    m, n, k = shape
    tile_rows, splits, stages = plan(m, n, k, _abi.VDK_BF16 if dt == "bf16" else _abi.VDK_FP32)
    assert tile_rows == tile and (splits > 1) == shared
    if two is not None:
        assert (stages < DEEP[tile]) == two
    share = -(-k // 128) // splits
    assert share > stages, "a turn of the ring"
    assert (share > SCALE_BLOCKS[tile]) == (shape not in ONE_CHUNK), "a chunk of scales"
    g = gen(m + n + k)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    bias = randn(g, n) if m % 2 else None
    ref, mag = linear_ref(a, sa, w, sw, bias)
    out = ops.fp8_linear(a, sa, w, sw, bias=bias, out_dtype=DT[dt])
    ops.check_status()
    within(out, ref, linear_bound(mag, ref, k, DT[dt]))
    # The same rows by themselves: another tile's neighbours do not matter, and the sums have one order.
    again = ops.fp8_linear(a, sa, w, sw, bias=bias, out_dtype=DT[dt])
    assert torch.equal(again, out)


def test_the_plan_names_the_kernel_for_many_rows():
    assert plan(8192, 24576, 4096)[0] == 0 and plan(515, 6144, 4096)[0] == 0
    assert plan(1, 1, 1)[:2] == (16, 1)
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 1 << 31)):
        with pytest.raises(_abi.VdError):
            plan(*bad)
    with pytest.raises(_abi.VdError):
        plan(1, 1, 1, 3)
