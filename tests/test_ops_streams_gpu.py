"""One context's calls on several streams of the caller's."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
TENSOR = 2


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    yield o
    o.close()


def gemm_case(seed, n=256, k=4096, rows=32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w, x = (torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16) for shape in ((n, k), (rows, k)))
    y = torch.zeros(rows, n, dtype=torch.bfloat16, device="cuda")
    return w, x, y


def alone(ops, case):
    """What the call gives by itself."""
    w, x, y = case
    torch.cuda.synchronize()
    ops.stream()
    ops.gemm(w, x, y, TENSOR, 8)
    ops.sync()
    want = y.clone()
    # a sum of k products in f32, in pieces: every addition off by 2^-23 of the magnitudes at most; one rounding
    mag = x.double().abs() @ w.double().abs().T
    exact = x.double() @ w.double().T
    assert ((want.double() - exact).abs() <= exact.abs() * 2.0 ** -8 + w.shape[1] * 2.0 ** -23 * mag).all()
    y.zero_()
    torch.cuda.synchronize()
    return want


@pytest.mark.parametrize("call", ["gemm", "chain_gemm"])
@pytest.mark.parametrize("then", ["another stream", "the context's own"])
def test_scratch_is_used_by_one_call_at_a_time(ops, call, then):
    """A GEMM on one stream does not begin while one on another stream, behind a long kernel, has the scratch still to come."""
    a, b = gemm_case(1), gemm_case(2)
    if call == "gemm":
        want = alone(ops, a), alone(ops, b)
    go = (lambda c: ops.gemm(*c, TENSOR, 8)) if call == "gemm" else (lambda c: ops.chain_gemm(*c))
    go(a), ops.sync()  # whatever a first call sets up
    if call != "gemm":
        go(b), ops.sync()
        want = a[2].clone(), b[2].clone()
        a[2].zero_(), b[2].zero_()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        torch.cuda._sleep(400_000_000)  # 0.2 s and more
        ops.stream(s1.cuda_stream)
        go(a)
    ops.stream(s2.cuda_stream) if then == "another stream" else ops.stream()
    go(b)
    if then == "another stream":
        time.sleep(0.05)
        assert not s1.query(), "the long kernel was too short for the test"
        assert not s2.query(), "ran beside a call that uses the same scratch"
    else:
        ops.sync()
        assert s1.query(), "ran beside a call that uses the same scratch"
    torch.cuda.synchronize()
    ops.stream()
    ops.sync()
    assert torch.equal(a[2], want[0]) and torch.equal(b[2], want[1])


def test_split_gemms_in_turns_on_three_streams(ops):
    cases = [gemm_case(s, n, k) for s, (n, k) in enumerate([(256, 4096), (1024, 2048), (128, 8192), (512, 4096)])]
    want = [alone(ops, c) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), None]
    for turn in range(40):
        for i, c in enumerate(cases):
            s = streams[(turn + i) % 3]
            ops.stream(None if s is None else s.cuda_stream)
            ops.gemm(*c, TENSOR, 8)
        torch.cuda.synchronize()
        for c, w in zip(cases, want):
            assert torch.equal(c[2], w)
            c[2].zero_()
        torch.cuda.synchronize()
    ops.stream()
    ops.sync()


def test_scratch_is_not_captured(ops):
    """Two graphs that shared it could be replayed side by side: refused, and the capture goes on."""
    from pega_omni_b200.ops import OpsError
    w, x, y = gemm_case(5)
    qk = torch.randn(4, 3 * 64, device="cuda").to(torch.bfloat16)
    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 2 * 64, dtype=torch.bfloat16, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        ops.stream(stream.cuda_stream)
        for call in (lambda: ops.gemm(w, x, y, TENSOR, 8), lambda: ops.chain_gemm(w, x, y)):
            with pytest.raises(OpsError, match="captured"):
                call()
        ops.qk_norm_rope(qk, None, None, pos, 1, 1, 64, 1e-6, 1e4, out)
    ops.stream()
    graph.replay()
    torch.cuda.synchronize()
    assert out.abs().sum() > 0 and (y == 0).all()
    ops.gemm(w, x, y, TENSOR, 8)
    ops.sync()
    assert y.abs().sum() > 0
