"""fp8_linear writes nothing beside its output, whatever the last columns are and wherever the rows lie."""

import pytest

torch = pytest.importorskip("torch")

from test_operators_gpu import DT, gen, linear_bound, linear_ref, operand, within  # noqa: E402
from verdict_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu


# Rows by which each kernel is taken: few, up to 128 and many.
@pytest.mark.parametrize("m", [3, 50, 100, 129, 600])
@pytest.mark.parametrize("n", [5, 13, 120, 121, 127, 129, 489, 1141, 1144])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_nothing_beside_the_output_is_written(m, n, dt):
    k = 200
    g = gen(m * n)
    a, sa = operand(g, m, k, 1)
    w, sw = operand(g, n, k, 128)
    ref, mag = linear_ref(a, sa, w, sw, None)
    bound = linear_bound(mag, ref, k, DT[dt])
    unit = 16 // torch.empty(0, dtype=DT[dt]).element_size()
    # Rows on 16-byte boundaries with little and much room behind them, rows side by side, and rows off the boundary.
    for ld, first in ((-(-n // unit) * unit, unit), (-(-n // unit) * unit + 2 * unit, 0), (n, 0), (n + 1, 1)):
        size = first + (m - 1) * ld + n
        buf = torch.full((size + 64,), 7.0, device="cuda", dtype=DT[dt])
        out = buf.as_strided((m, n), (ld, 1), first)
        ops.fp8_linear(a, sa, w, sw, out_dtype=DT[dt], out=out)
        within(out, ref, bound)
        out.fill_(7.0)
        assert (buf == 7).all(), (ld, first)
