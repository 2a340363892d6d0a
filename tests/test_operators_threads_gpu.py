"""The 8-bit decoder operators called from threads that have made no CUDA call before."""

import threading

import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [5, 100, 600])
def test_a_product_is_a_threads_first_call(m):
    g = torch.Generator(device="cuda").manual_seed(m)
    a = ops.quantize_fp8(torch.randn(m, 1024, generator=g, device="cuda"))
    w = ops.quantize_fp8_weight(torch.randn(2048, 1024, generator=g, device="cuda"))
    want = ops.fp8_linear(*a, *w)
    torch.cuda.synchronize()
    got, failed = [], []

    def worker():
        try:
            got.append(ops.fp8_linear(*a, *w))
        except Exception as e:
            failed.append(e)

    t = threading.Thread(target=worker)
    t.start()
    t.join(60)
    assert not failed, failed
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)
