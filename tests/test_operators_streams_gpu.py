"""The 8-bit decoder operators run on the stream that is current: their inputs change in stream order, and an operator
that ran elsewhere, or in a graph on copies, would read the values before the change."""

import math

import pytest

torch = pytest.importorskip("torch")

from verdict_b200 import ops  # noqa: E402

pytestmark = pytest.mark.gpu

F8 = ops.FP8


def prepare():
    g = torch.Generator(device="cuda").manual_seed(11)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w, sw = ops.quantize_fp8_weight(rand(1024, 512) * 0.05)
    gain = 1 + 0.1 * rand(512)
    plan = ops.RotaryPlan(64)
    x, h, pos = rand(20, 512).to(torch.bfloat16), rand(20, 512), torch.arange(20, device="cuda")
    real = (x, h, pos)
    other = ((2 * rand(20, 512)).to(torch.bfloat16), rand(20, 512), pos * 37 + 5)
    bufs = [t.clone() for t in real]

    def chain():
        x, h, pos = bufs
        cast = ops.quantize_fp8(x, gate=x, act="silu")
        r = ops.block_norm(x, h, post_gain=gain, pre_gain=gain, out_dtype=F8)
        o = ops.fp8_linear(r.out, r.scale, w, sw)
        q, _ = ops.rotary(o.view(20, 16, 64), None, pos, plan)
        lp = ops.token_logprobs(q.reshape(20, 1024), pos[:, None], top=3)
        weight = ops.quantize_fp8_weight(x)
        return [cast[0].float(), cast[1], r.residual, r.out.float(), r.scale, o, q, lp.logprobs, lp.entropy, lp.lse,
                lp.top_ids, weight[0].float(), weight[1]]

    def put(values):
        for b, v in zip(bufs, values):
            b.copy_(v)

    def answers(values):
        put(values)
        out = [t.clone() for t in chain()]
        torch.cuda.synchronize()
        return out

    return chain, put, answers(real), answers(other), real, other, bufs


def same(got, want):
    return [torch.equal(a, b) for a, b in zip(got, want)]


def test_operators_wait_for_what_the_current_stream_writes():
    chain, put, want, others, real, other, bufs = prepare()
    assert not any(same(want, others))
    for b in bufs[:2]:
        b.fill_(math.nan)
    bufs[2].fill_(7)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # ten milliseconds, in which only the stale values are there
        put(real)
        got = chain()
    side.synchronize()
    assert all(same(got, want)), same(got, want)


def test_a_graph_reads_its_inputs_when_it_is_replayed():
    chain, put, want, others, real, other, _ = prepare()
    put(real)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for values, expected in ((other, others), (real, want), (other, others)):
        put(values)
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(got, expected)), same(got, expected)
    # On another stream, after the change queued there.
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        put(real)
        graph.replay()
    side.synchronize()
    assert all(same(got, want)), same(got, want)
    ops.check_status()


@pytest.mark.parametrize("m,n,k", [(3, 4096, 512), (100, 4096, 2048), (600, 4096, 512)])
def test_a_product_reads_what_the_product_before_it_wrote(m, n, k):
    """Each of these kernels is set up while the two before it still run.  A buffer that the first reads as its bias, the
    second writes as its output and the third reads as its bias again must not come out of a cache."""
    g = torch.Generator(device="cuda").manual_seed(m)
    a = ops.quantize_fp8(torch.randn(m, k, generator=g, device="cuda"))
    w = ops.quantize_fp8_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    one = ops.quantize_fp8(torch.randn(1, k, generator=g, device="cuda"))
    start = torch.randn(n, generator=g, device="cuda")

    def chain(wait):
        bias, out = start.clone(), torch.empty(m, n, device="cuda")
        results = []
        for _ in range(20):
            results.append(ops.fp8_linear(*a, *w, bias=bias, out_dtype=torch.float32))   # reads the bias
            wait()
            ops.fp8_linear(*one, *w, out_dtype=torch.float32, out=bias.view(1, n))        # writes it
            wait()
            ops.fp8_linear(*a, *w, bias=bias, out_dtype=torch.float32, out=out)           # reads it again
            wait()
            results.append(out.clone())
            bias.copy_(start)
        return results

    want = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert all(same(chain(lambda: None), want))


def test_products_of_every_kind_on_several_streams_at_once():
    """CTAs of different products meet on an SM and share its tensor memory; the answers are those of one at a time."""
    g = torch.Generator(device="cuda").manual_seed(9)
    work = []
    for m, n, k in ((3, 512, 32768), (16, 24576, 1024), (30, 512, 32768), (50, 4096, 12288), (64, 20000, 1024),
                    (100, 4096, 12288), (100, 3000, 300), (600, 2048, 4096)):
        a = ops.quantize_fp8(torch.randn(m, k, generator=g, device="cuda"))
        w = ops.quantize_fp8_weight(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
        work.append((a, w))
    logits = torch.randn(4, 152064, generator=g, device="cuda")
    run = lambda i: ops.fp8_linear(*work[i][0], *work[i][1])  # noqa: E731
    want = [run(i) for i in range(len(work))]
    want_lp = ops.token_logprobs(logits, top=5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got, got_lp = [], []
    for rounds in range(12):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for j in range(len(work)):
                    i = (j * (2 * s + 1) + rounds + s) % len(work)
                    got.append((i, run(i)))
                got_lp.append(ops.token_logprobs(logits, top=5))
    torch.cuda.synchronize()
    ops.check_status()
    assert all(torch.equal(t, want[i]) for i, t in got)
    assert all(torch.equal(a, b) for r in got_lp for a, b in zip(r[1:], want_lp[1:]))
