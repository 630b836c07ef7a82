"""Decode attention over 8-bit pages with scores of any size: softmax looks at their differences alone."""
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


@pytest.mark.parametrize("hq,hk,d", [(2, 1, 128), (16, 1, 64), (9, 1, 128)])
@pytest.mark.parametrize("size", [0.0, 1.0, 3e3, 1e7, 3e8, 1e12, 1e25, 1e31, 2e37, -1.0, -3e3, -1e7, -3e8, -1e12, -1e25, -1e31, -2e37])
@pytest.mark.parametrize("t", [1, 5, 16, 40, 777, 9000])
def test_scores_of_any_size(ops, t, size, hq, hk, d):
    """Keys with one element, which is 2 or 1: scores are twice `size` or once, those of the smaller ones equal bit for bit. Some pages'
    values are 2^20 apart."""
    g = torch.Generator(device="cuda")
    g.manual_seed(t)
    n = -(-t // PAGE)
    vals = (torch.randn(n, hk, 2, PAGE, d, generator=g, device="cuda") * 90).clamp(-240, 240).to(torch.float8_e4m3fn).float()
    high = torch.rand(n * PAGE, generator=g, device="cuda") < 0.2
    vals[:, :, 0] = 0
    vals[:, :, 0, :, 0] = torch.where(high, 256.0, 128.0).view(n, 1, PAGE)
    kv = vals.to(torch.float8_e4m3fn)
    scales = torch.full((n, hk, 2), 2.0 ** -7, device="cuda")
    scales[::3, :, 1] = 2.0 ** 13
    q = torch.zeros(1, hq, d, device="cuda")
    q[:, :, 0] = size
    q = q.to(torch.bfloat16)
    x = kv.double() * scales.double()[..., None, None]
    k, v = (x[:, :, i].transpose(0, 1).reshape(hk, -1, d)[:, :t].repeat_interleave(hq // hk, 0) for i in (0, 1))
    # one product a score, and the scale: two roundings of it, which are the same for equal keys
    s = (k[:, :, 0] * q[0, :, 0, None].double()) * 0.5
    w = torch.softmax(s, -1)
    want = (w[:, None] @ v)[:, 0]
    # where both kinds count, their difference is off by 3 roundings of a score; the weights' to f16: 2^-11 of itself or 2^-16 of the page's
    # largest; ex2 and sums over t tokens; the result's rounding
    r = (3 * 2.0 ** -23 * s.abs().amax() if abs(size) < 1e4 else 0) + 2.0 ** -11 + 2.0 ** -22 + (t / 2 + 8) * 2.0 ** -23
    pages = torch.nn.functional.pad(w, (0, n * PAGE - t)).view(hq, -1, PAGE).amax(-1).repeat_interleave(PAGE, -1)[:, :t]
    tol = want.abs() * 2.0 ** -8 + ((w * 2 * r + pages * 2.0 ** -16)[:, None] @ v.abs())[:, 0] * (1 + 2.0 ** -7) + 1e-30
    out = torch.empty(1, hq * d, dtype=torch.bfloat16, device="cuda")
    ops.kv8_attend(q.view(1, hq * d), kv.view(torch.uint8), scales, i32([t - 1]), i32([0, n]), i32(np.arange(n)), hq, 0.5, out)
    ops.sync()
    off = (out.double().view_as(want) - want).abs() / tol
    assert off.max() <= 1, off.max().item()
