"""Decode attention over 8-bit pages where nearly all of a row's weight lies on tokens without a value: what is left is the result."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def ops(built_lib):
    from pega_omni_b200.ops import Ops
    o = Ops(0)
    o.stream(0)  # tensors of these tests live on the default stream
    yield o
    o.close()


def i32(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


def check(ops, hq, hk, d, loud, rest, seed=0):
    """One row per entry of `loud`, which marks the tokens that have no value and, together, 1 / rest times the weight of the others."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    scale, lens = 0.125, [len(m) for m in loud]
    counts = [-(-t // PAGE) for t in lens]
    total, indptr = sum(counts), np.concatenate([[0], np.cumsum(counts)])
    codes = (torch.randn(total, hk, 2, PAGE, d, generator=g, device="cuda") * 90).clamp(-240, 240).to(torch.float8_e4m3fn)
    scales = torch.full((total, hk, 2), 2.0 ** -7, device="cuda")
    vals = codes.float()
    vals[:, :, 0, :, 0] = 0  # a key's first element is what makes it loud, and all that it has
    for n, m in enumerate(loud):
        at = torch.zeros(counts[n], PAGE, dtype=torch.bool, device="cuda")
        at.view(-1)[:lens[n]] = torch.from_numpy(m).cuda()
        part = vals[indptr[n]:indptr[n + 1]]
        part[:] = torch.where(at[:, None, None, :, None], 0, part)
        part[:, :, 0, :, 0] = torch.where(at[:, None], 256.0, 0.0)
    kv = vals.to(torch.float8_e4m3fn)
    assert torch.equal(kv.float(), vals)
    q = (torch.randn(len(loud), hq, d, generator=g, device="cuda") / (scale * 0.7 * d ** 0.5)).to(torch.bfloat16)
    x = kv.double() * scales.double()[..., None, None]
    want, tol = (torch.zeros(len(loud), hq, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for n, t in enumerate(lens):
        k, v = (x[indptr[n]:indptr[n + 1], :, i].transpose(0, 1).reshape(hk, -1, d)[:, :t].repeat_interleave(hq // hk, 0) for i in (0, 1))
        m = torch.from_numpy(loud[n]).cuda()
        s = (k @ q[n].double()[..., None])[..., 0] * scale
        others = torch.logsumexp(torch.where(m, -float("inf"), s), -1)
        q[n, :, 0] = (others - np.log(rest) - np.log(m.sum().item())) / (2.0 * scale)  # a loud key's first element is 2
        s = (k @ q[n].double()[..., None])[..., 0] * scale
        w = torch.softmax(s, -1)
        assert torch.where(m, w, 0).sum(-1).min() > 1 - 3 * rest
        want[n] = (w[:, None] @ v)[:, 0]
        # a weight's rounding to f16: 2^-11 of itself or 2^-16 of its page's largest, or 2^-60 of the row's largest; the rest as for any
        # other row: scores are sums of d products, every addition off by 2^-23 of the magnitudes at most, scaled by products of f32
        # (another 4); ex2 and the f32 sums over t tokens; the result's rounding
        top = torch.nn.functional.pad(w, (0, counts[n] * PAGE - t)).view(hq, -1, PAGE).amax(-1).repeat_interleave(PAGE, -1)[:, :t]
        off = torch.maximum(w * 2.0 ** -11, top * 2.0 ** -16) + w.amax(-1, keepdim=True) * 2.0 ** -60
        mag = (k.abs() @ q[n].double().abs()[..., None]).amax(1) * scale
        r = 2 * (d + 4) * 2.0 ** -23 * mag + (t / 2 + 8) * 2.0 ** -23
        tol[n] = want[n].abs() * 2.0 ** -8 + ((off + w * r)[:, None] @ v.abs())[:, 0] * (1 + 2.0 ** -7) + 1e-38
    out = torch.empty(len(loud), hq * d, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q.view(len(loud), hq * d), kv.view(torch.uint8), scales, i32([t - 1 for t in lens]), i32(indptr), i32(np.arange(total)), hq, scale, out)
    ops.sync()
    off = (out.double().view_as(want) - want).abs() / tol
    assert off.max() <= 1, off.max().item()


def sink(t, at):
    m = np.zeros(t, dtype=bool)
    m[at] = True
    return m


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 128), (16, 1, 128), (20, 4, 64), (16, 1, 64)])
@pytest.mark.parametrize("rest", [1e-2, 1e-3, 1e-5, 1e-8, 1e-12])
@pytest.mark.parametrize("t,at", [(300, 0), (4000, 0), (4000, 1234), (4000, 3999), (60000, 0), (60000, 59999)])
def test_a_sink_without_a_value(ops, t, at, rest, hq, hk, d):
    """A token that has the weight, first, last or between, in rows of a CTA, of a cluster and in pieces."""
    check(ops, hq, hk, d, [sink(t, at)], rest, seed=t + at)


@pytest.mark.parametrize("rest", [1e-3, 1e-8])
def test_sinks_of_many_rows(ops, rest):
    """Enough rows that each has CTAs of its own, of all lengths."""
    rng = np.random.default_rng(5)
    lens = rng.integers(20, 900, 200)
    check(ops, 4, 2, 128, [sink(t, rng.integers(0, t)) for t in lens], rest, seed=5)


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("rest", [1e-1, 1e-3, 1e-4, 1e-5, 1e-6, 1e-9, 1e-15])
@pytest.mark.parametrize("every", [2, 3, 9])
def test_loud_and_quiet_pages_in_turns(ops, every, rest, hq, hk, d):
    """References that go up and down from page to page."""
    t = 3000
    check(ops, hq, hk, d, [np.arange(t) // PAGE % every == 0, np.arange(t) // PAGE % every == every - 1], rest, seed=every)
