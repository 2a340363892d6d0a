"""Types and shapes of the 8-bit decoder operators that the first tests leave out."""

import pytest

torch = pytest.importorskip("torch")

from test_operators_gpu import (DT, F8, HALF_ULP, NORM_REL, TINY, U, blocks_of, dequant, gen, norm_ref, randn,  # noqa: E402
                                strided, within)
from verdict_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,cols,pad,offset", [(1, 1, 0, 0), (129, 127, 0, 0), (257, 384, 8, 0), (300, 1001, 3, 1)])
def test_quantize_weight_in_every_type(rows, cols, pad, offset, dt):
    w = randn(gen(rows + cols), rows, cols, dtype=DT[dt])
    w[0, 0] = 0
    w[:min(rows, 128), :min(cols, 128)] *= 0 if cols == 384 else 1  # a block of zeros
    q, s = ops.quantize_fp8_weight(strided(w, pad, offset))
    nr, nc = -(-rows // 128), -(-cols // 128)
    assert q.shape == w.shape and s.shape == (nr, nc) and (q.shape[0] == 1 or q.stride(0) % 16 == 0)
    f = torch.zeros(nr * 128, nc * 128, device="cuda")
    f[:rows, :cols] = w.float()
    b = f.view(nr, 128, nc, 128)
    amax = b.abs().amax((1, 3)).clamp_min(1e-30)
    limit = torch.full_like(amax, 448.0)
    assert torch.equal(s, amax / limit)
    want = (b * (limit / amax)[:, None, :, None]).clamp(-448, 448).to(F8).float().reshape(nr * 128, nc * 128)
    assert torch.equal(q.float(), want[:rows, :cols])


@pytest.mark.parametrize("tokens,heads", [(1, 40), (77, 8), (515, 12)])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("plus_one", [False, True])
def test_block_norm_on_the_rows_of_heads(tokens, heads, hd, dt, plus_one):
    """What q and k get before their rotary positions: a norm over each head."""
    g = gen(tokens + hd)
    x = randn(g, tokens * heads, hd, dtype=DT[dt], scale=2.0)
    gain = 1 + randn(g, hd, scale=0.1)
    _, mag, z = norm_ref(None, x, None, None, 1.0, 1.0, gain, 1e-6, plus_one)
    zerr = 4 * NORM_REL * z.abs()
    for view in (x, strided(x, 3)):
        r = ops.block_norm(None, view, pre_gain=gain, plus_one=plus_one)
        assert r.residual is view and r.out.dtype == DT[dt]
        within(r.out, z, zerr + HALF_ULP[DT[dt]] * z.abs() + TINY[DT[dt]])
    r = ops.block_norm(None, x, pre_gain=gain, plus_one=plus_one, out_dtype=F8)
    amax = blocks_of(z, lambda c: c.abs().amax(1))
    within(r.scale, amax / 448, (4 * NORM_REL + 2 * U) * amax / 448)
    sc = r.scale.double().repeat_interleave(128, 1)[:, :hd]
    within(dequant(r.out, r.scale), z, torch.maximum(z.abs() * 2.0 ** -4, sc * 2.0 ** -10) * (1 + 1e-3) + 2 * zerr)
