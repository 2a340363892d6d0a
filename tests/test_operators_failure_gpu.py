"""fp8_linear where a pipeline wait runs out, without a GPU fault.

The stall is made on purpose and stays in bounds: each CTA loads its first few
k-blocks (valid tiles) and then stops, so its other warps wait for a stage that
nothing will fill; a short limit ends that wait.  The kernel has to return, to
leave the wait's code in the status word and to leave the context usable.
"""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import _abi, ops  # noqa: E402

pytestmark = pytest.mark.gpu

# One shape per kernel: up to 16, 32, 64 and 128 rows a tile with K split over a cluster and not, CTA pairs.
SHAPES = [(3, 512, 32768), (3, 24576, 4096), (30, 512, 32768), (50, 512, 16384), (60, 20000, 4096), (100, 4096, 12288),
          (600, 2048, 16384)]


def operands(m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a = ops.quantize_fp8(torch.randn(m, k, generator=g, device="cuda"))
    w = ops.quantize_fp8_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    return a, w


def limited(a, w, out, status, limit_us, stall_after):
    (q, s), (wq, ws) = a, w
    err = ctypes.create_string_buffer(512)
    rc = _abi.load().vdk_fp8_linear_stalled(
        q.data_ptr(), q.stride(0), s.data_ptr(), s.stride(0), wq.data_ptr(), wq.stride(0), ws.data_ptr(), ws.stride(0),
        q.shape[0], wq.shape[0], q.shape[1], None, out.data_ptr(), out.stride(0), _abi.VDK_BF16, status.data_ptr(),
        limit_us, stall_after, torch.cuda.current_stream().cuda_stream, err, 512)
    _abi.check(rc, err)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_a_stalled_product_returns_and_says_so(m, n, k):
    a, w = operands(m, n, k)
    want = ops.fp8_linear(*a, *w)
    out = torch.empty_like(want)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    # Nothing loaded; one block; a chunk of scales exactly (8 or 16 blocks), one less and one more; past a ring.
    for stall_after in (0, 1, 2, 7, 8, 9, 15, 16, 17):
        if stall_after * 128 >= k // 8:  # the smallest share of K that a CTA may have
            continue
        status.zero_()
        limited(a, w, out, status, 1000, stall_after)
        torch.cuda.synchronize()
        assert int(status) != 0, stall_after
        # The context and the SMs' tensor memory are as before.
        assert torch.equal(ops.fp8_linear(*a, *w), want), stall_after
    ops.check_status()


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_a_short_limit_alone_changes_nothing(m, n, k):
    a, w = operands(m, n, k)
    want = ops.fp8_linear(*a, *w)
    out = torch.empty_like(want)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    limited(a, w, out, status, 100000, -1)
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(out, want)


def test_check_status_raises_once():
    a, w = operands(5, 256, 1024)
    want = ops.fp8_linear(*a, *w)
    limited(a, w, torch.empty_like(want), ops._status_word(want.device), 1000, 0)
    with pytest.raises(_abi.VdError) as e:
        ops.check_status()
    assert e.value.code == _abi.VD_ECUDA
    ops.check_status()
    assert torch.equal(ops.fp8_linear(*a, *w), want)


def test_every_thread_that_ran_products_learns_of_a_failure():
    import threading
    a, w = operands(5, 256, 1024)
    want = ops.fp8_linear(*a, *w)
    ran, go, told = threading.Barrier(3), threading.Barrier(3), []

    def worker(slot):
        ops.fp8_linear(*a, *w)
        ran.wait(60)
        go.wait(60)
        try:
            ops.check_status()
        except _abi.VdError:
            told.append(slot)
        ops.check_status()  # once

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    ran.wait(60)
    limited(a, w, torch.empty_like(want), ops._status_word(want.device), 1000, 0)
    with pytest.raises(_abi.VdError):
        ops.check_status()  # this thread asks first
    go.wait(60)
    for t in threads:
        t.join(60)
    assert sorted(told) == [0, 1]
    # A thread that starts afterwards has nothing to learn.
    late = []

    def newcomer():
        try:
            ops.fp8_linear(*a, *w)
            ops.check_status()
        except _abi.VdError as e:
            late.append(e)

    t = threading.Thread(target=newcomer)
    t.start()
    t.join(60)
    assert not late
    ops.check_status()
